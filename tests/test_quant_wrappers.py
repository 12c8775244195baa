"""What the Python calls of the quantised operators refuse before anything is launched, and whose memory they use."""
import pytest
import torch


def test_rows_that_overlap_have_no_stride(gsv):
    from gsv_b200 import quant

    assert quant._row_stride(torch.zeros(1, 8).expand(1, 8), "x") == 8
    assert quant._row_stride(torch.zeros(4, 12)[:, :8], "x") == 12
    for t in (torch.zeros(8).expand(4, 8), torch.zeros(40).as_strided((4, 8), (7, 1))):
        with pytest.raises(ValueError, match="overlap"):
            quant._row_stride(t, "x")


@pytest.mark.gpu
def test_expanded_tensors_are_refused(dev):
    """A broadcast row, weight or residual: its stride of 0 must not reach the C ABI."""
    x = torch.zeros(64, device="cuda")
    a = torch.zeros(4, 64, dtype=torch.int8, device="cuda")
    s = torch.ones(64, device="cuda")
    wide, wide8 = x.expand(4, 64), a[0].expand(4, 64)
    for call in (lambda: dev.quantize_rows_i8(wide), lambda: dev.quantize_rows_i8(wide.half()[:1].expand(4, 64)),
                 lambda: dev.quantize_rows_i8(x.repeat(4, 1), q=wide8), lambda: dev.gemm_i8(wide8, s, a, s),
                 lambda: dev.gemm_i8(a, s, wide8, s), lambda: dev.gemm_i8(a, s, a, s, residual=x[:4].expand(4, 4)),
                 lambda: dev.gemm_i8(a, s, a, s, residual=x[:1].expand(4, 4)),
                 lambda: dev.gemm_i8(a, s, a, s, c=x[:4].expand(4, 4)),
                 lambda: dev.gemm_i8(a, s, a, s, c_f16=x[:4].half().expand(4, 4))):
        with pytest.raises(ValueError):
            call()
    # one row has no stride
    assert dev.gemm_i8(a[:1].expand(1, 64), s, a, s, residual=x[:4].expand(1, 4)).shape == (1, 4)
