"""Rows in 8 bits that stand far apart: a place in them passes 32 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("m", [2, 3])
def test_quantised_rows_with_a_stride_beyond_an_int(m):
    from mimirmind_b200.kernels import ops
    gen = torch.Generator(device=DEV).manual_seed(m)
    k, n, stride = 400, 96, 2 ** 31 + 16
    w = ops.quantize_fp8_weight(0.05 * torch.randn((n, k), generator=gen, device=DEV))
    w_in, w_out = (ops.quantize_fp8_weight(0.05 * torch.randn(s, generator=gen, device=DEV)) for s in ((2, 144, k), (k, 144)))
    rows = ops.quantize_fp8_rows(torch.randn((m, k), generator=gen, device=DEV))
    wide = torch.empty((m - 1) * stride + 416, dtype=torch.uint8, device=DEV).as_strided((m, k), (stride, 1))
    wide.copy_(rows.values.view(torch.uint8))
    far = ops.Fp8Rows(wide.view(torch.float8_e4m3fn), rows.scales)
    assert far.ld == stride
    assert torch.equal(ops.gemm_fp8(far, w), ops.gemm_fp8(rows, w))
    assert torch.equal(ops.glu_mlp_fp8(far, w_in, w_out), ops.glu_mlp_fp8(rows, w_in, w_out))
