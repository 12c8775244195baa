"""The 8-bit integer linear layer at the ends of its number ranges: scales in fp32's subnormal range, infinities and NaN
through the activations, sizes past what a launch holds."""
import numpy as np
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("top", [3e-37, 1e-38, 4e-39, 1e-39, 1e-40])
@pytest.mark.parametrize("rows,n,pad", [(1, 8, 0), (3, 512, 0), (700, 512, 0), (2000, 512, 0), (5, 1024, 8), (64, 4096, 0),
                                        (3, 333, 0), (2, 20001, 7), (9, 1001, 3)])
def test_rows_whose_scale_has_no_finite_inverse(dev, rows, n, pad, top):
    rng = np.random.default_rng(n)
    x = (rng.uniform(-1, 1, (rows, n + pad)) * top).astype(np.float32)
    x[:, 3] = top
    x[-1] *= 1e30  # beside a row of ordinary size
    s = np.abs(x[:, :n]).max(1) / np.float32(127)
    want = np.rint(x[:, :n] / s[:, None]).astype(np.int8)
    for _ in range(4):
        q, scale = dev.quantize_rows_i8(torch.from_numpy(x).cuda()[:, :n])
        np.testing.assert_array_equal(scale.cpu().numpy(), s)
        np.testing.assert_array_equal(q.cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,pad", [(1, 8, 0), (700, 512, 0), (5, 1024, 8), (64, 4096, 0), (2, 20001, 7), (9, 1001, 3)])
def test_codes_stop_at_127(dev, rows, n, pad):
    """Near the smallest subnormals a scale is a few units of its last place, and x / scale passes 127: 190 units over 127
    are 1.496, a scale of 1."""
    tiny = np.finfo(np.float32).smallest_subnormal
    rng = np.random.default_rng(n)
    x = rng.integers(-190, 191, (rows, n + pad)).astype(np.float32) * tiny
    x[:, 2], x[:, n - 1] = 190 * tiny, -190 * tiny
    s = np.abs(x[:, :n]).max(1) / np.float32(127)
    assert (s == tiny).all()
    q, scale = dev.quantize_rows_i8(torch.from_numpy(x).cuda()[:, :n])
    np.testing.assert_array_equal(scale.cpu().numpy(), s)
    np.testing.assert_array_equal(q.cpu().numpy(), np.clip(np.rint(x[:, :n] / tiny), -127, 127).astype(np.int8))


def _both_paths(dev, a, b, sa, sb, **kw):
    """The product of rows in whole 16 bytes (tensor cores) and of the same rows an odd stride apart (CUDA cores)."""
    out = []
    for odd in (0, 1):
        t = []
        for x in (a, b):
            wide = torch.zeros(x.shape[0], x.shape[1] + odd, dtype=torch.int8, device="cuda")
            wide[:, :x.shape[1]] = x
            t.append(wide[:, :x.shape[1]])
        c = torch.empty(a.shape[0], b.shape[0], device="cuda")
        h = torch.empty_like(c, dtype=torch.float16)
        dev.gemm_i8(t[0], sa, t[1], sb, c=c, c_f16=h, **kw)
        out.append((c, h))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("act", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("M,N,K", [(70, 70, 64), (300, 520, 256), (1, 33, 16)])
def test_both_paths_give_the_same_bits(dev, M, N, K, act):
    gen = torch.Generator().manual_seed(act + M)
    a, b = (torch.randint(-127, 128, (r, K), generator=gen, dtype=torch.int8).cuda() for r in (M, N))
    sa, sb = (torch.rand(r, generator=gen).mul(0.03).cuda() for r in (M, N))
    bias, res = torch.randn(N, generator=gen).cuda(), torch.randn(M, N, generator=gen).cuda()
    bias[0], bias[-1], sa[M // 2] = float("inf"), float("-inf"), float("nan")
    for kw in (dict(), dict(residual=res)):
        (c0, h0), (c1, h1) = _both_paths(dev, a, b, sa, sb, bias=bias, act=act, slope=0.1, **kw)
        for x, y in ((c0, c1), (h0, h1)):
            np.testing.assert_array_equal(x.cpu().numpy(), y.cpu().numpy())


@pytest.mark.gpu
def test_gelu_at_the_infinities(dev):
    """x Phi(x): inf at inf, 0 at -inf and far below 0, NaN for NaN; what is large and finite stays."""
    one = torch.ones(4, device="cuda")
    a, b = torch.zeros(4, 16, dtype=torch.int8, device="cuda"), torch.zeros(8, 16, dtype=torch.int8, device="cuda")
    inf = float("inf")
    bias = torch.tensor([inf, -inf, float("nan"), 3e38, -3e38, 1e20, -1e20, 0.0], device="cuda")
    want = np.array([inf, 0, np.nan, 3e38, 0, 1e20, 0, 0], np.float32)
    for c, _ in _both_paths(dev, a, b, one, torch.ones(8, device="cuda"), bias=bias, act=2):
        np.testing.assert_array_equal(c.cpu().numpy(), np.tile(want, (4, 1)))


@pytest.mark.gpu
@pytest.mark.parametrize("act", [0, 1, 2, 3, 4])
def test_a_bad_row_shows_through_every_activation(dev, act):
    """The scale of a row with a NaN or an infinity is NaN: no activation may make an ordinary row of it."""
    x = torch.randn(40, 96, generator=torch.Generator().manual_seed(3)).half().cuda()
    x[7, 3], x[9, 0] = float("nan"), float("inf")
    w, ws = dev.quantize_rows_i8(torch.randn(50, 96, generator=torch.Generator().manual_seed(4)).cuda())
    q, s = dev.quantize_rows_i8(x)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[7, 9]] = True
    for c, h in _both_paths(dev, q, w, s, ws, act=act, slope=0.1):
        for y in (c, h):
            assert y[bad].isnan().all() and y[~bad].isfinite().all()


@pytest.mark.parametrize("M,N", [(2**31 - 300, 2**31 - 300), (2**30, 2**30), (2**25, 2**24), (2**20 + 1, 2**19)])
def test_more_outputs_than_a_launch_holds_are_refused(gsv, M, N):
    """A block count past 32 bits must not wrap to a small grid."""
    import ctypes

    from gsv_b200.quant import GemmI8Args

    for ld in (64, 65):
        g = GemmI8Args(a=256, lda=ld, b=256, ldb=ld, a_scale=256, b_scale=256, M=M, N=N, K=64, c=256, ldc=N)
        assert gsv.lib().gsvk_gemm_i8(ctypes.byref(g), None) == -5


def test_the_packed_gelu_has_gelu_erfs_constants():
    """The polynomial of Phi(-u) stands in both sources, two values to an operation in the product's: the same numbers."""
    import os
    import re

    src = os.path.join(os.path.dirname(__file__), "..", "gpt-sovits-native_b200", "csrc")

    def body(name, start):
        text = open(os.path.join(src, name)).read()
        text = text[text.index(start):]
        return text[:text.index("\n}\n")]

    scalar = re.findall(r"[-+]?\d\.\d+e[-+]\d+f", body("common.cuh", "float gelu_erf(float x)"))
    packed = re.findall(r"pair\(([-+]?\d\.\d+e[-+]\d+f), ([-+]?\d\.\d+e[-+]\d+f)\)", body("gemm_i8.cu", "void gelu2("))
    assert len(scalar) == 11 and packed == [(c, c) for c in scalar]
    for text in (body("common.cuh", "float gelu_erf(float x)"), body("gemm_i8.cu", "void gelu2(")):
        assert "-0.721347520444f" in text and "5.5f" in text
