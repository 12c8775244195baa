"""The T2S decoder stack over the paged 4-bit cache and the 8-bit linear layers, against the same layers in 64 bits.

The plain stack quantises where the served one does (kv4_ref.quantise, rows to int8 over max / 127) and computes in fp64,
so the two differ where a code falls on the other side of a tie.  The served rows between operators are fp16 or fp32, off
by up to 2^-11 of themselves: an int8 step is max / 127 > 2^-7 of the row's rms, so a few codes in a hundred move by one,
rms below sqrt(0.06) * 0.028 = 0.7 % of a row; a 4-bit step is half the rms, so a code in a thousand moves, 1.6 %; and as
much again in the tokens after them, by way of the cache.  With four products and a cache a layer, two layers and three
steps, whose errors add like a random walk and which the LayerNorms keep in proportion: below sqrt(2 * (4 * 0.7^2 + 2 *
1.6^2)) = 3.8 % rms, 5 % with what earlier steps left.  A missing prefix, a wrong slot, layer or residual moves rows by
tens of per cent (checked below, on the plain side)."""
import numpy as np
import pytest

import kv4_ref as ref

BOUND = 0.05


def _model(gsv, seed, d_model=128, heads=4, ffn=256, vocab=65):
    m = gsv.workloads.t2s_model(n_layers=2, d_model=d_model, n_heads=heads, ffn=ffn, vocab=vocab, seed=seed)
    for name in ("wqkv", "wout", "w1", "w2", "wpred"):  # scores of unit variance: attention that matters
        w = m[name].view(np.float16).astype(np.float32)
        m[name] = np.ascontiguousarray((w / (0.02 * np.sqrt(w.shape[-1]))).astype(np.float16)).view(np.uint16)
    return m


def _int8(x):
    x = x.astype(np.float32)
    s = np.abs(x).max(-1, keepdims=True) / np.float32(127)
    return np.rint(x / s).astype(np.float64) * s.astype(np.float64)


def _linear(x, w, b=0.0):
    return _int8(x) @ _int8(w.view(np.float16)).T + b


def _norm(x, g, b, eps):
    d = x - x.mean(-1, keepdims=True)
    return d / np.sqrt((d * d).mean(-1, keepdims=True) + eps) * g + b


class Plain:
    """Requests one after the other, each with its own unpaged lists of quantised rows."""

    def __init__(self, m, n_seq):
        self.m = m
        self.kv = [[[] for _ in range(m["n_layers"])] for _ in range(n_seq)]

    def step(self, i, x, prefix, wrong=None):
        """x [rows, d_model] of request i."""
        m, H = self.m, self.m["n_heads"]
        hd = m["d_model"] // H
        n = len(x)
        for l in range(m["n_layers"]):
            qkv = _linear(x, m["wqkv"][l], m["bqkv"][l]).astype(np.float16).reshape(n, 3, H, hd)
            kv = self.kv[i][0 if wrong == "layer" else l]
            kv += [[ref.values(*ref.quantise(t)) for t in row[1:]] for row in qkv]
            K, V = np.array([r[0] for r in kv]), np.array([r[1] for r in kv])
            s = np.einsum("thd,jhd->htj", qkv[:, 0].astype(np.float64), K) / np.sqrt(hd)
            total = len(kv)
            limit = np.minimum(total, np.maximum(prefix, total - n + np.arange(n) + 1))
            s = np.where(np.arange(total) < limit[:, None], s, -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            y = np.einsum("htj,jhd->thd", p / p.sum(-1, keepdims=True), V).reshape(n, -1)
            x = _norm(x + _linear(y, m["wout"][l], m["bout"][l]), m["n1g"][l], m["n1b"][l], m["ln_eps"])
            f = np.maximum(_linear(x, m["w1"][l], m["b1"][l]), 0)
            x = _norm(x + _linear(f, m["w2"][l], m["b2"][l]), m["n2g"][l], m["n2b"][l], m["ln_eps"])
        return x


def _off(a, b):
    return float(np.sqrt(((a - b) ** 2).mean() / (b ** 2).mean()))


# rows of each request, step by step (prompts of 40, 1, 70 and none; then single tokens beside a late prompt)
STEPS = [[40, 1, 70, 0], [1, 1, 1, 33], [1, 0, 1, 1]]
PREFIX = [16, 0, 70, 5]


def _run_plain(m, xs, wrong=None):
    plain, out = Plain(m, 4), []
    for rows, x in zip(STEPS, xs):
        at = np.concatenate([[0], np.cumsum(rows)])
        out.append(np.concatenate([plain.step(i, x[at[i]:at[i + 1]].astype(np.float64),
                                              0 if wrong == "prefix" else PREFIX[i], wrong)
                                   for i in range(4) if rows[i]]))
    return out


def _inputs(seed, d_model=128):
    rng = np.random.default_rng(seed)
    return [rng.standard_normal((sum(r), d_model), dtype=np.float32) for r in STEPS]


@pytest.mark.parametrize("wrong", ["prefix", "layer"])
def test_the_bound_tells_a_wrong_stack(gsv, wrong):
    m, xs = _model(gsv, 3), _inputs(4)
    good, bad = _run_plain(m, xs), _run_plain(m, xs, wrong)
    assert max(_off(b, a) for a, b in zip(good, bad)) > 3 * BOUND


@pytest.mark.gpu
@pytest.mark.parametrize("page,d_model,heads", [(16, 128, 4), (64, 128, 2), (32, 256, 2)])
def test_steps_of_prompts_and_tokens(dev, page, d_model, heads):
    import torch

    m, xs = _model(dev, 3, d_model=d_model, heads=heads), _inputs(4, d_model)
    t2s = dev.T2SPaged(m, max_seq=4, max_tokens=128, max_len=128, n_pages=4 * (128 // page), page_size=page)
    prefix = torch.tensor(PREFIX, dtype=torch.int32, device="cuda")
    for rows, x, want in zip(STEPS, xs, _run_plain(m, xs)):
        new = torch.tensor(rows, dtype=torch.int32, device="cuda")
        got = t2s.step(torch.from_numpy(x).cuda(), new, max_q=max(rows), prefix=prefix)
        assert int(t2s.plan.refused) == 0
        assert _off(got.double().cpu().numpy(), want) < BOUND
        last = np.cumsum(rows)[[i for i in range(4) if rows[i]]] - 1
        logits = t2s.logits(got).double().cpu().numpy()[[i for i in range(4) if rows[i]]]
        assert _off(logits, _linear(want[last], m["wpred"])) < BOUND
    assert t2s.length.tolist() == [42, 2, 72, 34]
    held = 4 * (128 // page) - int(t2s.free_count)
    assert held == sum(-(-n // page) for n in t2s.length.tolist())
    t2s.release(torch.tensor([1, 1, 0, 1], dtype=torch.int32, device="cuda"))
    assert t2s.length.tolist() == [0, 0, 72, 0]
    assert int(t2s.free_count) == 4 * (128 // page) - -(-72 // page)


@pytest.mark.gpu
def test_a_place_is_used_again(dev):
    """A request that takes the pages of one that left sees none of its rows."""
    import torch

    m, xs = _model(dev, 5), _inputs(6)
    new = torch.tensor(STEPS[0], dtype=torch.int32, device="cuda")
    x = torch.from_numpy(xs[0]).cuda()
    t2s = dev.T2SPaged(m, max_seq=4, max_tokens=128, max_len=128, n_pages=9, page_size=16)
    first = t2s.step(x, new, max_q=70)
    t2s.release(torch.ones(4, dtype=torch.int32, device="cuda"))
    assert torch.equal(t2s.step(x, new, max_q=70), first)


@pytest.mark.gpu
def test_decoding_replays_from_a_graph(dev):
    """Greedy tokens of captured steps are those of single calls."""
    import torch

    m = _model(dev, 7)
    xs = torch.from_numpy(_inputs(8)[0]).cuda()
    new = torch.tensor(STEPS[0], dtype=torch.int32, device="cuda")
    ones = torch.tensor([1, 1, 1, 0], dtype=torch.int32, device="cuda")
    pick = torch.tensor([0, 1, 2], device="cuda")

    def start():
        t2s = dev.T2SPaged(m, max_seq=4, max_tokens=128, max_len=128, n_pages=32, page_size=16)
        return t2s, t2s.greedy(t2s.step(xs, new, max_q=70))[pick], t2s.length[pick].clone()

    def decode(t2s, tok, pos):
        tok.copy_(t2s.greedy(t2s.step(t2s.embed(tok, pos), ones, max_q=1))[pick])
        pos.add_(1)

    t2s, tok, pos = start()
    want = []
    for _ in range(6):
        decode(t2s, tok, pos)
        want.append(tok.tolist())
    assert int(t2s.plan.refused) == 0

    t2s, tok, pos = start()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    with torch.cuda.stream(side):
        decode(t2s, tok, pos)
        got.append(tok.tolist())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decode(t2s, tok, pos)
    for _ in range(5):
        graph.replay()
        got.append(tok.tolist())
    assert got == want


@pytest.mark.gpu
def test_a_full_pool_refuses(dev):
    import torch

    m = _model(dev, 9)
    t2s = dev.T2SPaged(m, max_seq=2, max_tokens=64, max_len=64, n_pages=2, page_size=16)
    x = torch.randn(48, m["d_model"], device="cuda")
    t2s.step(x, torch.tensor([20, 28], dtype=torch.int32, device="cuda"), max_q=28)
    assert int(t2s.plan.refused) == 1 and t2s.length.tolist() == [20, 0]
    with pytest.raises(ValueError):
        t2s.step(torch.randn(65, m["d_model"], device="cuda"), torch.tensor([1, 64], dtype=torch.int32, device="cuda"), 64)
