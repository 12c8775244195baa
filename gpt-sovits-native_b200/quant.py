"""Quantised serving: the paged 4-bit KV cache (page plan, append, read back,
attention) and the 8-bit integer linear layer, over the C ABI of
include/gsvk.h, which states the value rules and the page layout.

A decode step of many requests is

    plan.run(ctx_len, new_len, table, free, free_count)      # pages and slots, on the GPU
    for each layer:
        codes, s = quantize_rows_i8(x)
        qkv = gemm_i8(codes, s, wqkv, wqkv_scale, bias)
        cache.append(k, v, plan.slots)
        y = cache.attention(q, plan.q_start, plan.kv_len, table, scale, max_q, workspace=ws)

Every call is asynchronous on its stream and runs on the current device, where
its tensors have to be; objects here hold device buffers and must not be used
from two streams at once.
"""
from __future__ import annotations

import ctypes
from ctypes import byref, c_float, c_int, c_size_t, c_void_p

from . import ACT_NONE, check, lib

_vp, _sz = c_void_p, c_size_t


class KVPlanArgs(ctypes.Structure):
    _fields_ = [("n_seq", _sz), ("max_blocks", _sz), ("n_pages", _sz), ("max_tokens", _sz),
                ("page_size", c_int), ("ctx_len", _vp), ("new_len", _vp), ("block_table", _vp),
                ("free_pages", _vp), ("free_count", _vp), ("q_start", _vp), ("kv_len", _vp),
                ("slots", _vp), ("free_left", _vp), ("refused", _vp), ("workspace", _vp)]


class KV4CacheArgs(ctypes.Structure):
    _fields_ = [("pages", _vp), ("n_pages", _sz), ("page_size", c_int), ("kv_heads", c_int),
                ("head_dim", c_int)]


class KV4AttentionArgs(ctypes.Structure):
    _fields_ = [("cache", KV4CacheArgs), ("q", _vp), ("q_stride", _sz), ("out", _vp),
                ("out_stride", _sz), ("heads", _sz), ("n_tokens", _sz), ("n_seq", _sz),
                ("max_blocks", _sz), ("max_q", _sz), ("q_start", _vp), ("kv_len", _vp),
                ("prefix", _vp), ("block_table", _vp), ("scale", c_float), ("workspace", _vp),
                ("workspace_bytes", _sz)]


class GemmI8Args(ctypes.Structure):
    _fields_ = [("a", _vp), ("lda", _sz), ("b", _vp), ("ldb", _sz), ("a_scale", _vp),
                ("b_scale", _vp), ("M", _sz), ("N", _sz), ("K", _sz), ("bias", _vp),
                ("residual", _vp), ("ld_res", _sz), ("c", _vp), ("ldc", _sz), ("c_f16", _vp),
                ("ldc_f16", _sz), ("act", c_int), ("slope", c_float)]


_current = None


def _device():
    """Index of the current device, None without one.  The C ABI launches there,
    so that is where every tensor and stream of a call has to be."""
    global _current
    if _current is None:
        import torch

        _current = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
    try:
        return _current()
    except RuntimeError:
        return None


def _home(index, what):
    """Index of the current device, where an object that holds memory has to have it."""
    here = _device()
    if index != here:
        raise ValueError(f"{what}: on cuda:{index}, the current device is cuda:{here}")
    return here


def _device_for(device):
    """The current device, which a `device` that is given has to be."""
    import torch

    current = torch.device("cuda", torch.cuda.current_device())
    if device is not None:
        device = torch.device(device)
        if device.type != "cuda" or device.index not in (None, current.index):
            raise ValueError(f"device: {device} is not the current device {current}")
    return current


_raw_stream = None


def _stream_for(stream, here):
    """Handle of `stream`, or of the current stream of the current device `here`.
    At a decode step's sizes a call takes a few microseconds, which making a
    Stream object (torch.cuda.current_stream) would double: torch's raw handle
    is read instead where it is to be had."""
    global _raw_stream
    if stream is not None:
        index = getattr(stream, "device_index", here)
        if index != here:
            raise ValueError(f"stream: of cuda:{index}, the current device is cuda:{here}")
        return stream.cuda_stream
    if _raw_stream is None:
        import torch

        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                              lambda device: torch.cuda.current_stream(device).cuda_stream)
    return _raw_stream(here)


def _on_device(t, what, here):
    """Refuses a tensor that is not on the current device `here`."""
    if not t.is_cuda:
        raise ValueError(f"{what}: gsvk takes CUDA tensors")
    if t.get_device() != here:
        raise ValueError(f"{what}: on cuda:{t.get_device()}, the current device is cuda:{here}")


def _tensor(t, dtype, dim, what, here):
    """Address of a CUDA tensor of one type and rank whose rows are contiguous."""
    if (t.dtype is dtype and t.get_device() == here and t.dim() == dim
            and (t.stride(-1) == 1 or t.shape[-1] < 2)):
        return t.data_ptr()
    _on_device(t, what, here)
    if t.dtype is not dtype:
        raise TypeError(f"{what}: {dtype} expected, got {t.dtype}")
    if t.dim() != dim:
        raise ValueError(f"{what}: {dim} dimensions expected, got {t.dim()}")
    raise ValueError(f"{what}: gsvk takes tensors with unit inner stride")


def _vector(t, dtype, n, what, here):
    """Address of at least n contiguous values."""
    if t.dtype is dtype and t.get_device() == here and t.is_contiguous() and t.numel() >= n:
        return t.data_ptr()
    _on_device(t, what, here)
    if t.dtype is not dtype:
        raise TypeError(f"{what}: {dtype} expected, got {t.dtype}")
    raise ValueError(f"{what}: {n} contiguous values expected")


def _row_stride(t, rows, n, what):
    """Elements between the rows of a tensor [rows, n] (one row: any), which may
    not overlap: to the C ABI the stride 0 of an expanded tensor means dense
    rows."""
    if rows < 2:
        return n
    ld = t.stride(0)
    if ld < n:
        raise ValueError(f"{what}: rows of {n} values, {ld} apart, overlap")
    return ld


def _rows(t, dtype, heads, head_dim, what, here):
    """Address and row stride of [tokens, heads, head_dim] rows whose heads lie side by side."""
    p = _tensor(t, dtype, 3, what, here)
    n, h, d = t.shape
    if h != heads or d != head_dim:
        raise ValueError(f"{what}: [tokens, {heads}, {head_dim}] expected, got {tuple(t.shape)}")
    row, head, _ = t.stride()
    if heads > 1 and head != head_dim:
        raise ValueError(f"{what}: the heads of a row lie side by side")
    return p, row if n > 1 else heads * head_dim


def _allocator(stream):
    """Where a call's outputs come from: torch.empty, or for a call on a stream
    that is given, that stream's own memory (the current one's may still be in
    use by work that is queued there), kept by the allocator until the current
    stream, whose it is to read, is done with it too."""
    import torch

    if stream is None:
        return torch.empty

    def empty(shape, dtype, device):
        with torch.cuda.stream(stream):
            t = torch.empty(shape, dtype=dtype, device=device)
        t.record_stream(torch.cuda.current_stream(device))
        return t

    return empty


def _hold(stream, *tensors):
    """Memory that a call on a stream that is given uses is its owner's to give
    up at once, and the allocator's to keep until the call has run."""
    for t in tensors:
        if t is not None:
            t.record_stream(stream)


def _filled():
    """Waits for the fills of an object's own buffers, which calls on any stream
    may then use: the caller has no other handle on them.  (A capture orders
    its own.)"""
    import torch

    if not torch.cuda.is_current_stream_capturing():
        torch.cuda.current_stream().synchronize()


# ------------------------------------------------------------------ page plan
class KVPlan:
    """Pages and slots of each step of up to `n_seq` requests, built on the GPU
    (gsvk_kv_plan).  Holds the results: q_start, kv_len, slots, free_left,
    refused."""

    def __init__(self, n_seq: int, max_blocks: int, page_size: int, n_pages: int, max_tokens: int,
                 device=None):
        import torch

        device = _device_for(device)
        i32 = dict(dtype=torch.int32, device=device)
        self.n_seq, self.max_blocks, self.n_pages = int(n_seq), int(max_blocks), int(n_pages)
        self.page_size, self.max_tokens = int(page_size), int(max_tokens)
        self._table_shape, self._index = (self.n_seq, self.max_blocks), device.index
        self.q_start = torch.zeros(n_seq + 1, **i32)
        self.kv_len = torch.zeros(n_seq, **i32)
        self.slots = torch.full((max_tokens,), -1, dtype=torch.int64, device=device)
        self.free_left = torch.zeros(1, **i32)
        self.refused = torch.zeros(1, **i32)
        self._ticket = torch.zeros(1, **i32)
        self._args = KVPlanArgs(
            n_seq=self.n_seq, max_blocks=self.max_blocks, n_pages=self.n_pages,
            max_tokens=self.max_tokens, page_size=self.page_size, q_start=self.q_start.data_ptr(),
            slots=self.slots.data_ptr(), refused=self.refused.data_ptr(),
            workspace=self._ticket.data_ptr())
        _filled()

    def _state(self, length, block_table, free_pages, free_count):
        import torch

        i32, here = torch.int32, _home(self._index, "the plan")
        if block_table.shape != self._table_shape:
            raise ValueError(f"block_table: {self._table_shape} expected, got "
                             f"{tuple(block_table.shape)}")
        return (here, _vector(length, i32, self.n_seq, "lengths", here),
                _vector(block_table, i32, 0, "block_table", here),
                _vector(free_pages, i32, self.n_pages, "free_pages", here),
                _vector(free_count, i32, 1, "free_count", here))

    def run(self, ctx_len, new_len, block_table, free_pages, free_count, in_place=False,
            stream=None):
        """Plans one step: `ctx_len` cached and `new_len` new tokens of each
        request (int32), the block table [n_seq, max_blocks], and the pool's
        free_pages[: free_count].  in_place: ctx_len and free_count become the
        lengths and the count after the step (and stand for kv_len and
        free_left), else those go to this object's own."""
        import torch

        a = self._args
        here, a.ctx_len, a.block_table, a.free_pages, a.free_count = self._state(
            ctx_len, block_table, free_pages, free_count)
        a.new_len = _vector(new_len, torch.int32, self.n_seq, "new_len", here)
        a.kv_len = a.ctx_len if in_place else self.kv_len.data_ptr()
        a.free_left = a.free_count if in_place else self.free_left.data_ptr()
        check(lib().gsvk_kv_plan(byref(a), _stream_for(stream, here)))
        if stream is not None:
            _hold(stream, ctx_len, new_len, block_table, free_pages, free_count, self.q_start,
                  self.kv_len, self.slots, self.free_left, self.refused, self._ticket)
        return self

    def release(self, done, length, block_table, free_pages, free_count, stream=None):
        """Returns the pages of the requests with done != 0 to the pool (in place)."""
        import torch

        here, ln, table, free, count = self._state(length, block_table, free_pages, free_count)
        check(lib().gsvk_kv_release(self.n_seq, self.max_blocks, self.n_pages, self.page_size,
                                    _vector(done, torch.int32, self.n_seq, "done", here), ln, table,
                                    free, count, _stream_for(stream, here)))
        if stream is not None:
            _hold(stream, done, length, block_table, free_pages, free_count)


# ------------------------------------------------------------- 4-bit KV cache
def kv4_page_bytes(page_size: int, kv_heads: int, head_dim: int) -> int:
    """Bytes of a page; 0 where the sizes are not supported."""
    return lib().gsvk_kv4_page_bytes(page_size, kv_heads, head_dim)


class KV4Workspace:
    """Scratch of KV4Cache.attention for up to `n_seq` requests and `n_tokens`
    rows; the layers of a model share one, as may models of any head_dim whose
    calls do not overlap.  After a device-side wait that ran out
    (device_status) its buffer has to be zeroed."""

    def __init__(self, n_seq: int, n_tokens: int, heads: int, kv_heads: int, head_dim: int,
                 device=None):
        import torch

        device = _device_for(device)
        self.index = device.index
        self.bytes = lib().gsvk_kv4_attention_workspace(n_seq, n_tokens, heads, kv_heads, head_dim)
        if self.bytes == 0:
            raise ValueError(f"no attention for {n_seq} requests, {n_tokens} rows, {heads} heads "
                             f"over {kv_heads} of {head_dim}")
        self.buffer = torch.zeros(self.bytes, dtype=torch.uint8, device=device)
        self.ptr = self.buffer.data_ptr()
        _filled()


class KV4Cache:
    """One layer's pages: a uint8 CUDA tensor [n_pages, kv4_page_bytes(...)]."""

    def __init__(self, pages, page_size: int, kv_heads: int, head_dim: int):
        import torch

        size = kv4_page_bytes(page_size, kv_heads, head_dim)
        if size == 0:
            raise ValueError(f"no 4-bit cache with pages of {page_size} tokens, {kv_heads} heads "
                             f"of {head_dim}")
        p = _vector(pages, torch.uint8, size, "pages", _device())
        if pages.numel() % size:
            raise ValueError(f"pages: whole pages of {size} bytes expected")
        self.pages, self._index = pages, pages.get_device()
        self.page_size, self.kv_heads, self.head_dim = int(page_size), int(kv_heads), int(head_dim)
        self.n_pages = pages.numel() // size
        self._cache = KV4CacheArgs(p, self.n_pages, self.page_size, self.kv_heads, self.head_dim)
        self._attn = KV4AttentionArgs(cache=self._cache)
        self._ref, self._attn_ref = byref(self._cache), byref(self._attn)

    @classmethod
    def empty(cls, n_pages: int, page_size: int, kv_heads: int, head_dim: int, device=None):
        import torch

        size = kv4_page_bytes(page_size, kv_heads, head_dim)
        pages = torch.empty(n_pages, max(size, 1), dtype=torch.uint8, device=_device_for(device))
        return cls(pages, page_size, kv_heads, head_dim)

    def append(self, k, v, slots, stream=None):
        """Quantises rows [tokens, kv_heads, head_dim] (fp16 or fp32) into their
        slots (int64; those outside the cache, such as -1, are skipped)."""
        import torch

        dtype, here = v.dtype, _home(self._index, "the cache")
        if dtype is not torch.float16 and dtype is not torch.float32:
            raise TypeError(f"k, v: fp16 or fp32 expected, got {dtype}")
        kp, ks = _rows(k, dtype, self.kv_heads, self.head_dim, "k", here)
        vp, vs = _rows(v, dtype, self.kv_heads, self.head_dim, "v", here)
        n = k.shape[0]
        if v.shape[0] != n:
            raise ValueError(f"k, v: {n} and {v.shape[0]} rows")
        check(lib().gsvk_kv4_append(self._ref, kp, ks, vp, vs, dtype is torch.float32,
                                    _vector(slots, torch.int64, n, "slots", here), n,
                                    _stream_for(stream, here)))
        if stream is not None:
            _hold(stream, k, v, slots, self.pages)

    def read(self, slots, k=None, v=None, stream=None):
        """What the slots stand for: fp16 rows k and v [len(slots), kv_heads,
        head_dim], zeros for a slot outside the cache."""
        import torch

        n, here = slots.numel(), _home(self._index, "the cache")
        sp = _vector(slots, torch.int64, n, "slots", here)
        if k is None and v is None:
            shape = (n, self.kv_heads, self.head_dim)
            empty = _allocator(stream)
            k = empty(shape, dtype=torch.float16, device=slots.device)
            v = torch.empty_like(k) if stream is None else empty(shape, torch.float16, slots.device)
        kp = ks = vp = vs = 0
        for t, what in ((k, "k"), (v, "v")):
            if t is not None and t.shape[0] != n:
                raise ValueError(f"{what}: {n} rows expected, got {t.shape[0]}")
        if k is not None:
            kp, ks = _rows(k, torch.float16, self.kv_heads, self.head_dim, "k", here)
        if v is not None:
            vp, vs = _rows(v, torch.float16, self.kv_heads, self.head_dim, "v", here)
        check(lib().gsvk_kv4_read(self._ref, sp, n, kp, ks, vp, vs, _stream_for(stream, here)))
        if stream is not None:
            _hold(stream, slots, k, v, self.pages)
        return k, v

    def attention(self, q, q_start, kv_len, block_table, scale: float, max_q: int, workspace,
                  prefix=None, out=None, stream=None):
        """Attention of packed rows q [tokens, heads, head_dim] (fp16) over the
        cache (gsvk_kv4_attention): request i owns rows q_start[i] to
        q_start[i + 1], sees kv_len[i] keys causally from the end and its
        first prefix[i] from every row.  `workspace`: a KV4Workspace of at
        least these sizes and of no smaller head_dim.  Returns fp16 rows like q."""
        import torch

        f16, i32, here = torch.float16, torch.int32, _home(self._index, "the cache")
        if q.dim() != 3:
            raise ValueError(f"q: [tokens, heads, {self.head_dim}] expected, got {tuple(q.shape)}")
        n, heads, _ = q.shape
        a = self._attn
        a.q, a.q_stride = _rows(q, f16, heads, self.head_dim, "q", here)
        if out is None:
            out = _allocator(stream)((n, heads, self.head_dim), dtype=f16, device=q.device)
            a.out, a.out_stride = out.data_ptr(), heads * self.head_dim
        else:
            if out.shape != q.shape:
                raise ValueError(f"out: {tuple(q.shape)} expected, got {tuple(out.shape)}")
            a.out, a.out_stride = _rows(out, f16, heads, self.head_dim, "out", here)
        if block_table.dim() != 2:
            raise ValueError(f"block_table: 2 dimensions expected, got {block_table.dim()}")
        n_seq, a.max_blocks = block_table.shape
        a.heads, a.n_tokens, a.n_seq, a.max_q, a.scale = heads, n, n_seq, max_q, scale
        a.q_start = _vector(q_start, i32, n_seq + 1, "q_start", here)
        a.kv_len = _vector(kv_len, i32, n_seq, "kv_len", here)
        a.prefix = None if prefix is None else _vector(prefix, i32, n_seq, "prefix", here)
        a.block_table = _vector(block_table, i32, 0, "block_table", here)
        if workspace.index != here:
            raise ValueError(f"workspace: on cuda:{workspace.index}, the current device is "
                             f"cuda:{here}")
        a.workspace, a.workspace_bytes = workspace.ptr, workspace.bytes
        check(lib().gsvk_kv4_attention(self._attn_ref, _stream_for(stream, here)))
        if stream is not None:
            _hold(stream, q, q_start, kv_len, prefix, block_table, out, workspace.buffer,
                  self.pages)
        return out


# -------------------------------------------------------- 8-bit linear layers
def quantize_rows_i8(x, q=None, scale=None, stream=None):
    """Rows of x [rows, n] (fp16 or fp32) as int8 codes and an fp32 scale each.
    A new q has its rows in whole 16 bytes, as gemm_i8's tensor-core path
    takes them."""
    import torch

    dtype, here = x.dtype, _device()
    if dtype is not torch.float16 and dtype is not torch.float32:
        raise TypeError(f"x: fp16 or fp32 expected, got {dtype}")
    xp = _tensor(x, dtype, 2, "x", here)
    rows, n = x.shape
    if q is None:
        ldq = (n + 15) & ~15
        q = _allocator(stream)((rows, ldq), dtype=torch.int8, device=x.device)
        qp = q.data_ptr()
        if ldq != n:
            q = q[:, :n]
    else:
        if q.shape != x.shape:
            raise ValueError(f"q: {(rows, n)} expected, got {tuple(q.shape)}")
        qp = _tensor(q, torch.int8, 2, "q", here)
        ldq = _row_stride(q, rows, n, "q")
    if scale is None:
        scale = _allocator(stream)(rows, dtype=torch.float32, device=x.device)
        sp = scale.data_ptr()
    else:
        sp = _vector(scale, torch.float32, rows, "scale", here)
    check(lib().gsvk_quantize_rows_i8(xp, dtype is torch.float32, rows, n,
                                      _row_stride(x, rows, n, "x"), qp, ldq, sp,
                                      _stream_for(stream, here)))
    if stream is not None:
        _hold(stream, x, q, scale)
    return q, scale


def gemm_i8(a, a_scale, b, b_scale, bias=None, residual=None, act=ACT_NONE, slope=0.0, c=None,
            c_f16=None, stream=None):
    """act(a_scale[m] b_scale[n] sum_k a[m, k] b[n, k] + bias) + residual: int8
    a [M, K] and b [N, K] -> fp32 c and / or fp16 c_f16 (a new fp16 one
    where neither is given)."""
    import torch

    i8, f32, here = torch.int8, torch.float32, _device()
    ap, bp = _tensor(a, i8, 2, "a", here), _tensor(b, i8, 2, "b", here)
    M, K = a.shape
    N, kb = b.shape
    if kb != K:
        raise ValueError(f"a, b: rows of {K} and {kb}")
    cp = ldc = hp = ldh = rp = ldr = 0
    if c is not None:
        cp, ldc = _matrix(c, f32, M, N, "c", here)
    if c_f16 is not None:
        hp, ldh = _matrix(c_f16, torch.float16, M, N, "c_f16", here)
    elif c is None:
        c_f16 = _allocator(stream)((M, N), dtype=torch.float16, device=a.device)
        hp, ldh = c_f16.data_ptr(), N
    if residual is not None:
        rp, ldr = _matrix(residual, f32, M, N, "residual", here)
    g = GemmI8Args(ap, _row_stride(a, M, K, "a"), bp, _row_stride(b, N, K, "b"),
                   _vector(a_scale, f32, M, "a_scale", here),
                   _vector(b_scale, f32, N, "b_scale", here), M, N, K,
                   None if bias is None else _vector(bias, f32, N, "bias", here), rp, ldr, cp,
                   ldc, hp, ldh, act, slope)
    check(lib().gsvk_gemm_i8(byref(g), _stream_for(stream, here)))
    if stream is not None:
        _hold(stream, a, a_scale, b, b_scale, bias, residual, c, c_f16)
    return c if c is not None else c_f16


def _matrix(t, dtype, M, N, what, here):
    """Address and row stride of an [M, N] tensor."""
    p = _tensor(t, dtype, 2, what, here)
    if t.shape[0] != M or t.shape[1] != N:
        raise ValueError(f"{what}: {(M, N)} expected, got {tuple(t.shape)}")
    return p, _row_stride(t, M, N, what)
