"""Hidden rows of the layer for a few tokens keep more bits than one 16-bit number has: seen where two of them nearly cancel."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [1, 3, 5, 16])
def test_hidden_rows_that_nearly_cancel(n, fp8):
    """The gate is 32 (silu(32) = 32 in fp32), the up projections are 128 + 2^-j and 128, the second matrix takes their difference: 32 * 2^-j, an exact number, where one
    number of 11 bits leaves nought for j > 4 (two bf16 parts keep j up to 9: 2^-17 of a number is lost)."""
    from mimirmind_b200.kernels import ops
    d, f = 128, 128
    x = torch.zeros((n, d), dtype=torch.bfloat16, device=DEV)
    x[:, :2] = 1.0
    w_in, w_out = torch.zeros((1, 2, f, d), device=DEV), torch.zeros((1, d, f), device=DEV)
    w_in[0, 0, :, 0] = 32.0
    w_in[0, 1, :, 0] = 128.0
    steps = [2.0 ** -j for j in range(4, 10)]
    for i, step in enumerate(steps):
        w_in[0, 1, 2 * i, 1] = step
        w_out[0, i, 2 * i], w_out[0, i, 2 * i + 1] = 1.0, -1.0
    if fp8:                                                   # scale 1
        def blocks(w):
            q = ops.fp8_weight_like(*w.shape, device=DEV)
            q.values.view(torch.uint8).copy_(w.to(torch.float8_e4m3fn).view(torch.uint8))
            q.scales.fill_(1.0)
            return q
        w_in, w_out = blocks(w_in), blocks(w_out)
    else:
        w_in, w_out = w_in.view(1, 2 * f, d).to(torch.bfloat16), w_out.to(torch.bfloat16)
    got = ops.moe_few(x, torch.zeros((1, d), device=DEV), w_in, w_out, 1)
    want = torch.zeros((n, d), device=DEV)
    want[:, :len(steps)] = 32.0 * torch.tensor(steps, device=DEV)
    assert torch.equal(got.float(), want)
