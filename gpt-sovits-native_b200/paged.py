"""The T2S decoder stack served from a paged 4-bit KV cache with 8-bit linear
layers: requests of any lengths join, decode and leave one shared pool of
pages, and a step takes prompts and single tokens side by side.

    t2s = T2SPaged(model, max_seq=64, max_tokens=4096, max_len=1600, n_pages=1600)
    x = t2s.step(rows, new_len, max_q=256, prefix=text_len)      # packed rows of every request
    tok = t2s.greedy(x)                                          # per request, from its last row
    while ...:
        tok = t2s.greedy(t2s.step(t2s.embed(tok, position), ones, max_q=1))
    t2s.release(done)

The layers are those of the T2S decoder (t2s_engine.cpp:1036-1118: fused QKV,
attention, output projection, LayerNorm, ReLU feed-forward, LayerNorm) and the
mask is its prefill's (t2s_engine.cpp:881-1034): the text prefix is seen by
every row, the rest causally.  The batched engine (T2SBatch) keeps a dense
fp16 cache per request and fp16 weights; this one trades their exactness
(cache rows in 4 bits, operands in 8) and some speed (1.62 ms a step of 64
requests of 529 tokens against 1.42) for 0.31 of the cache and half of the
weights.

A step makes no host read and leaves its lengths, tables and free pages on the
GPU, so a step of fixed row counts can be captured into a CUDA graph and
replayed.
"""
from __future__ import annotations

from . import ACT_RELU, layernorm_rows
from .quant import (KV4Cache, KV4Workspace, KVPlan, _device, _device_for, _row_stride, _tensor,
                    _vector, gemm_i8, quantize_rows_i8)


class Linear8:
    """A linear layer held as int8 rows with one scale each (the activations'
    rows are quantised at the call)."""

    def __init__(self, w, bias=None):
        self.codes, self.scale = quantize_rows_i8(w)
        self.bias = bias

    def __call__(self, x, **out):
        codes, scale = quantize_rows_i8(x)
        return gemm_i8(codes, scale, self.codes, self.scale, bias=self.bias, **out)


class T2SPaged:
    def __init__(self, model: dict, max_seq: int, max_tokens: int, max_len: int, n_pages: int,
                 page_size: int = 64, device=None):
        """`model`: as T2SBatch takes it.  Up to `max_seq` requests of up to
        `max_len` tokens, `max_tokens` packed rows a step, `n_pages` pages of
        `page_size` tokens in each layer's pool."""
        import numpy as np
        import torch

        device = _device_for(device)
        self.device, self.max_seq, self.max_tokens = device, int(max_seq), int(max_tokens)
        self.d_model, self.heads = model["d_model"], model["n_heads"]
        self.head_dim = self.d_model // self.heads
        self.eps = float(model["ln_eps"])
        self.scale = self.head_dim ** -0.5

        def put(a):
            a = np.ascontiguousarray(a)
            return torch.from_numpy(a.view(np.float16) if a.dtype == np.uint16 else a).to(device)

        self.layers = []
        for i in range(model["n_layers"]):
            self.layers.append(dict(
                qkv=Linear8(put(model["wqkv"][i]), put(model["bqkv"][i])),
                out=Linear8(put(model["wout"][i]), put(model["bout"][i])),
                up=Linear8(put(model["w1"][i]), put(model["b1"][i])),
                down=Linear8(put(model["w2"][i]), put(model["b2"][i])),
                norm1=(put(model["n1g"][i]), put(model["n1b"][i])),
                norm2=(put(model["n2g"][i]), put(model["n2b"][i])),
                cache=KV4Cache.empty(n_pages, page_size, self.heads, self.head_dim, device)))
        self.head = Linear8(put(model["wpred"]))
        self.audio_emb = put(model["audio_emb"]).float()
        self.alpha = float(model["alpha_audio"])
        self.freq = torch.exp(torch.arange(0, self.d_model, 2, device=device, dtype=torch.float32)
                              * np.float32(-np.log(10000.0) / self.d_model))
        i32 = dict(dtype=torch.int32, device=device)
        max_blocks = -(-int(max_len) // page_size)
        self.plan = KVPlan(self.max_seq, max_blocks, page_size, n_pages, self.max_tokens, device)
        self.workspace = KV4Workspace(self.max_seq, self.max_tokens, self.heads, self.heads,
                                      self.head_dim, device)
        self.length = torch.zeros(self.max_seq, **i32)
        self.block_table = torch.full((self.max_seq, max_blocks), -1, **i32)
        self.free_pages = torch.arange(n_pages, **i32)
        self.free_count = torch.full((1,), n_pages, **i32)

    def embed(self, tokens, positions):
        """Rows of audio tokens at their positions in the audio sequence
        (t2s_engine.cpp:1865-1869): embedding + alpha * sinusoid."""
        import torch

        angle = positions.float()[:, None] * self.freq
        pe = torch.stack([angle.sin(), angle.cos()], -1).view(len(tokens), self.d_model)
        return torch.add(self.audio_emb[tokens], pe, alpha=self.alpha)

    def step(self, x, new_len, max_q: int, prefix=None):
        """One step over packed rows x [tokens, d_model] (fp32): request i adds
        its new_len[i] rows (int32 CUDA, 0 for one that rests; their sum is
        the number of rows), none of them more than max_q.  `prefix`: leading
        tokens seen by every row of the request.  Returns the rows after the
        last layer; requests refused for want of pages are counted in
        self.plan.refused, keep their lengths, have -1 in self.plan.slots at
        their rows and get rows of no meaning."""
        import torch

        # all that a layer would refuse: the plan below moves the lengths on, so nothing may fail after it
        here = _device()
        _tensor(x, torch.float32, 2, "x", here)
        _row_stride(x, *x.shape, "x")
        if x.shape[1] != self.d_model:
            raise ValueError(f"x: rows of {self.d_model} expected, got {x.shape[1]}")
        n = x.shape[0]
        if n > self.max_tokens:
            raise ValueError(f"x: {n} rows in a step of up to {self.max_tokens}")
        if prefix is not None:
            _vector(prefix, torch.int32, self.max_seq, "prefix", here)
        plan = self.plan.run(self.length, new_len, self.block_table, self.free_pages,
                             self.free_count, in_place=True)
        if n == 0:  # every request rests
            return x
        for layer in self.layers:
            qkv = layer["qkv"](x).view(n, 3, self.heads, self.head_dim)
            layer["cache"].append(qkv[:, 1], qkv[:, 2], plan.slots)
            y = layer["cache"].attention(qkv[:, 0], plan.q_start, self.length, self.block_table,
                                         self.scale, max_q, self.workspace, prefix=prefix)
            y = layer["out"](y.view(n, self.d_model), residual=x, c=torch.empty_like(x))
            x = layernorm_rows(y, *layer["norm1"], self.eps)
            y = layer["down"](layer["up"](x, act=ACT_RELU), residual=x, c=torch.empty_like(x))
            x = layernorm_rows(y, *layer["norm2"], self.eps)
        return x

    def logits(self, x):
        """Logits (fp32) [max_seq, vocab] of each request's last row of a step;
        those of a request that had none are of no meaning.  x: at least one row."""
        import torch

        if len(x) == 0:  # the device would be asked for row 0 of none
            raise ValueError("x: no rows, so no logits")
        rows = x[(self.plan.q_start[1:] - 1).clamp(0, len(x) - 1).long()]
        return self.head(rows, c=torch.empty(self.max_seq, len(self.head.scale),
                                             dtype=torch.float32, device=self.device))

    def greedy(self, x):
        """Most likely token of each request after a step."""
        return self.logits(x).argmax(-1)

    def release(self, done):
        """Ends the requests with done != 0 (int32 CUDA): their pages return to
        the pool and their places are free."""
        self.plan.release(done, self.length, self.block_table, self.free_pages, self.free_count)
