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
