"""The 8-bit integer linear layer (gsvk_quantize_rows_i8, gsvk_gemm_i8): codes exactly, sums exactly, the epilogue
within its fp32 roundings."""
import ctypes
import math

import numpy as np
import pytest
import torch


def _quantise(x):
    x = x.astype(np.float32)
    with np.errstate(all="ignore"):
        top = np.abs(x).max(1)
        bad = ~np.isfinite(x).all(1)
        s = np.where(bad, np.float32(np.nan), top / np.float32(127))
        q = np.where((s > 0)[:, None], np.nan_to_num(np.rint(x / s[:, None])), 0)
    return np.where(bad[:, None], 0, q).astype(np.int8), s.astype(np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,n,pad", [(1, 1, 0), (1, 512, 0), (3, 17, 0), (64, 512, 1024), (33, 333, 0), (9, 1000, 24),
                                        (5, 4096, 0), (2, 20001, 7), (700, 768, 0)])
def test_codes_and_scales(dev, rows, n, pad, dtype):
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((rows, n + pad)) * rng.choice([1e-4, 1, 300], (rows, 1))).astype(dtype)
    x[0, :n] = (np.arange(n) % 255 - 127) * 0.5  # ties of the rounding
    if rows > 8:
        x[1], x[2, 0], x[3, n - 1], x[4, 0] = 0, np.nan, np.inf, -np.inf
        x[5, 0] = np.finfo(dtype).max
        x[6] = np.finfo(dtype).smallest_subnormal * 3
    t = torch.from_numpy(x).cuda()[:, :n]
    q, s = dev.quantize_rows_i8(t)
    wq, ws = _quantise(x[:, :n])
    np.testing.assert_array_equal(s.cpu().numpy(), ws)
    np.testing.assert_array_equal(q.cpu().numpy(), wq)
    # into the caller's rows: what lies between them stays
    own = torch.full((rows, n + 5), 99, dtype=torch.int8).cuda()
    dev.quantize_rows_i8(t, q=own[:, :n], scale=s)
    np.testing.assert_array_equal(own[:, :n].cpu().numpy(), wq)
    assert (own[:, n:] == 99).all()


def _operands(rng, M, N, K, lda, ldb):
    a = np.zeros((M, lda), np.int8)
    b = np.zeros((N, ldb), np.int8)
    a[:] = rng.integers(-128, 128, a.shape)
    b[:] = rng.integers(-128, 128, b.shape)
    sa = rng.uniform(0.5, 2, M).astype(np.float32) * 1e-2
    sb = rng.uniform(0.5, 2, N).astype(np.float32) * 1e-2
    ta, tb = torch.from_numpy(a).cuda()[:, :K], torch.from_numpy(b).cuda()[:, :K]
    return a[:, :K], b[:, :K], sa, sb, ta, tb, torch.from_numpy(sa).cuda(), torch.from_numpy(sb).cuda()


ACTS = {0: lambda y: y, 1: lambda y: np.maximum(y, 0), 3: lambda y: np.where(y < 0, y * 0.1, y), 4: np.tanh,
        2: lambda y: 0.5 * y * (1 + np.vectorize(math.erf)(y / math.sqrt(2)))}
SHAPES = [(1, 1, 1), (1, 1536, 512), (2, 7, 16), (5, 33, 40), (64, 1536, 512), (64, 1025, 512), (17, 129, 333),
          (100, 260, 2048), (128, 128, 128), (129, 255, 144), (300, 1025, 512), (256, 512, 1000), (513, 640, 256),
          (1000, 384, 4100), (16, 512, 8192), (257, 1, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("pad", ["whole", "odd"])
def test_product(dev, M, N, K, pad):
    """Every shape on rows of whole 16 bytes and on odd ones; the sum is exact, so the fp32 output differs from the
    64-bit one by the roundings of sa * sb, of the product's conversion and of the sum with the bias."""
    rng = np.random.default_rng(M * 3 + N + K)
    ld = (lambda k: k + -k % 16) if pad == "whole" else (lambda k: k + 1 + k % 2)
    a, b, sa, sb, ta, tb, tsa, tsb = _operands(rng, M, N, K, ld(K), ld(K) + (16 if pad == "whole" else 0))
    acc = a.astype(np.int64) @ b.astype(np.int64).T
    bias = rng.standard_normal(N).astype(np.float32)
    res = rng.standard_normal((M, N + 3)).astype(np.float32)
    y = acc * (sa.astype(np.float64)[:, None] * sb.astype(np.float64)) + bias.astype(np.float64)
    big = np.abs(acc * (sa.astype(np.float64)[:, None] * sb.astype(np.float64)))
    tol = 2**-22 * big + 2**-23 * np.abs(y) + 1e-30
    c = torch.full((M, N + 2), 5.0, device="cuda")
    h = torch.full((M, N + 1), 5.0, dtype=torch.float16, device="cuda")
    tbias, tres = torch.from_numpy(bias).cuda(), torch.from_numpy(res).cuda()
    dev.gemm_i8(ta, tsa, tb, tsb, bias=tbias, c=c[:, :N], c_f16=h[:, :N])
    got, got16 = c.cpu().numpy().astype(np.float64), h.cpu().numpy().astype(np.float64)
    assert (got[:, N:] == 5).all() and (got16[:, N:] == 5).all()
    assert (np.abs(got[:, :N] - y) <= tol).all()
    with np.errstate(over="ignore"):
        assert (got16[:, :N] == got[:, :N].astype(np.float32).astype(np.float16)).all()
    # with a residual that is the output itself
    r = tres[:, :N]
    dev.gemm_i8(ta, tsa, tb, tsb, residual=r, c=r)
    want = (y - bias) + res[:, :N]
    tol = 2**-21 * big + 2**-23 * np.abs(want) + 2**-23 * np.abs(res[:, :N]) + 1e-30
    got = tres.cpu().numpy().astype(np.float64)
    assert (np.abs(got[:, :N] - want) <= tol).all()
    np.testing.assert_array_equal(got[:, N:], res[:, N:])


@pytest.mark.gpu
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("M,N,K,ld", [(64, 200, 128, 128), (300, 300, 256, 256), (20, 50, 60, 61)])
def test_activations(dev, M, N, K, ld, act):
    rng = np.random.default_rng(act)
    a, b, sa, sb, ta, tb, tsa, tsb = _operands(rng, M, N, K, ld, ld)
    tsa *= 1e-2
    sa = tsa.cpu().numpy()
    bias = rng.standard_normal(N).astype(np.float32)
    x = (a.astype(np.int64) @ b.astype(np.int64).T) * (sa.astype(np.float64)[:, None] * sb) + bias
    got = dev.gemm_i8(ta, tsa, tb, tsb, bias=torch.from_numpy(bias).cuda(), act=act, slope=0.1)
    assert got.dtype == torch.float16
    want = ACTS[act](x)
    # the argument's fp32 error (slopes up to 1.13), the activation's own 4e-7, the rounding to fp16
    tol = 2**-11 * np.abs(want) + 2**-25 + 1.2 * 2**-21 * (np.abs(x) + np.abs(bias)) + 1e-6
    assert (np.abs(got.cpu().numpy().astype(np.float64) - want) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(3, 40), (300, 300)])
def test_sums_reach_the_end_of_32_bits(dev, M, N):
    """All codes -128 over the longest K: 2^31 - 2^14 is held exactly."""
    K = 131071
    a = torch.full((M, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    b = torch.full((N, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    one = torch.ones(max(M, N), device="cuda")
    c = torch.empty(M, N, device="cuda")
    dev.gemm_i8(a, one, b, one, c=c)
    assert (c == float(np.float32(K * 16384))).all()


@pytest.mark.gpu
def test_codes_between_k_and_the_leading_dimension_are_not_read(dev):
    a = torch.full((40, 64), 1, dtype=torch.int8, device="cuda")
    one = torch.ones(40, device="cuda")
    for K in (1, 15, 17, 33, 63):
        c = torch.empty(40, 40, device="cuda")
        dev.gemm_i8(a[:, :K], one, a[:, :K], one, c=c)
        assert (c == K).all()


@pytest.mark.gpu
def test_a_bad_row_stays_a_row(dev):
    """A NaN among the activations makes NaN of its token and of no other."""
    x = torch.randn(40, 96, device="cuda").half()
    w, ws = dev.quantize_rows_i8(torch.randn(50, 96, device="cuda"))
    clean = dev.gemm_i8(*dev.quantize_rows_i8(x), w, ws)
    x[7, 3], x[9, 0] = float("nan"), float("inf")
    got = dev.gemm_i8(*dev.quantize_rows_i8(x), w, ws)
    keep = [i for i in range(40) if i not in (7, 9)]
    assert got[[7, 9]].isnan().all() and torch.equal(got[keep], clean[keep])


@pytest.mark.gpu
def test_other_streams_and_empty_batches(dev):
    s = torch.cuda.Stream()
    x = torch.randn(70, 256, device="cuda").half()
    w, ws = dev.quantize_rows_i8(torch.randn(90, 256, device="cuda"))
    want = dev.gemm_i8(*dev.quantize_rows_i8(x), w, ws)
    s.wait_stream(torch.cuda.current_stream())
    q, sc = dev.quantize_rows_i8(x, stream=s)
    got = dev.gemm_i8(q, sc, w, ws, stream=s)
    s.synchronize()
    assert torch.equal(got, want)
    q, sc = dev.quantize_rows_i8(x[:0])
    assert q.shape == (0, 256) and dev.gemm_i8(q, sc, w, ws).shape == (0, 90)


@pytest.mark.gpu
def test_wrapper_checks(dev):
    a = torch.zeros(4, 32, dtype=torch.int8, device="cuda")
    s = torch.ones(4, device="cuda")
    for bad in (lambda: dev.gemm_i8(a, s, a[:, :16], s), lambda: dev.gemm_i8(a, s[:3], a, s),
                lambda: dev.gemm_i8(a, s, a, s, bias=s[:2]), lambda: dev.gemm_i8(a.t(), s, a, s),
                lambda: dev.gemm_i8(a, s, a, s, c=torch.zeros(4, 5, device="cuda")),
                lambda: dev.quantize_rows_i8(torch.zeros(4, device="cuda")),
                lambda: dev.quantize_rows_i8(a.float(), q=a[:2])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: dev.gemm_i8(a.float(), s, a, s), lambda: dev.gemm_i8(a, s.double(), a, s),
                lambda: dev.quantize_rows_i8(a)):
        with pytest.raises(TypeError):
            bad()


def _args(gsv, **over):
    from gsv_b200.quant import GemmI8Args

    g = dict(a=256, lda=64, b=256, ldb=64, a_scale=256, b_scale=256, M=4, N=8, K=64, c=256, ldc=8, act=0)
    g.update(over)
    return gsv.lib().gsvk_gemm_i8(ctypes.byref(GemmI8Args(**g)), None)


@pytest.mark.parametrize("over,rc", [(dict(a=None), -1), (dict(b=None), -1), (dict(a_scale=None), -1),
                                     (dict(b_scale=None), -1), (dict(c=None), -1), (dict(N=0), -1), (dict(K=0), -1),
                                     (dict(lda=63), -1), (dict(ldb=10), -1), (dict(ldc=7), -1), (dict(act=9), -1),
                                     (dict(K=131072, lda=0, ldb=0), -5), (dict(M=2**31), -5), (dict(N=2**40), -5),
                                     (dict(M=0), 0)])
def test_bad_arguments_are_refused_before_any_launch(gsv, over, rc):
    assert _args(gsv, **over) == rc


def test_bad_quantiser_arguments_are_refused_before_any_launch(gsv):
    q = gsv.lib().gsvk_quantize_rows_i8
    assert q(None, 0, 1, 4, 0, 256, 0, 256, None) == -1
    assert q(256, 0, 1, 0, 0, 256, 0, 256, None) == -1
    assert q(256, 0, 2, 8, 4, 256, 0, 256, None) == -1
    assert q(256, 0, 2, 8, 0, 256, 7, 256, None) == -1
    assert q(256, 0, 1, 2**31, 0, 256, 0, 256, None) == -5
    assert q(256, 0, 0, 8, 0, 256, 0, 256, None) == 0
