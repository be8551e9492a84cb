"""Hidden rows in 8 bits are e4m3(fl(h / s)): the quotient decides at the middle of two e4m3 numbers, where a product with fl(1 / s) falls to either side."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _middles():
    """(v, half a step) of 80 middles v + half a step of neighbouring e4m3 numbers; both are e4m3 numbers themselves"""
    pairs = [(2.0 ** e * (1 + m / 8), 2.0 ** (e - 4)) for e in range(-3, 9) for m in range(8)]
    return [p for p in pairs if sum(p) < 440][-80:]


def _feed_forward(d, factor):
    """A gate of 32 for every hidden column, an up projection of factor 256 (v + half a step) for column n, of factor 256 448 for column 80 and nought behind it; the second
    matrix hands the hidden columns on.  Products of powers of two and short numbers: every sum is one rounding, fl(factor (v + half a step))."""
    from mimirmind_b200.kernels import ops
    blocks = -(-d // 128)
    values = torch.zeros((2, 128, d), device=DEV)
    values[0, :, 0] = 32.0                                    # x 256, scale 2^-8: 32, whose silu is 32 in fp32
    for n, (v, half) in enumerate(_middles()):
        values[1, n, 0], values[1, n, 1] = v, half
    values[1, 80, 0] = 448.0
    scales = torch.ones((2, 1, blocks), device=DEV)
    scales[0] = 2.0 ** -8
    scales[1] = factor
    w_in = ops.fp8_weight_like(2, 128, d, device=DEV)
    w_in.values.view(torch.uint8).copy_(values.to(torch.float8_e4m3fn).view(torch.uint8))
    w_in.scales.copy_(scales)
    w_out = ops.quantize_fp8_weight(448.0 * torch.eye(128, device=DEV))           # scale 1
    w_out.values.view(torch.uint8).copy_(torch.eye(128, device=DEV).to(torch.float8_e4m3fn).view(torch.uint8))
    return w_in, w_out


@pytest.mark.parametrize("d", [128, 2048])
@pytest.mark.parametrize("m", [1, 12, 40, 200])
def test_hidden_rows_are_quotients(m, d):
    from mimirmind_b200.kernels import ops
    gen = torch.Generator().manual_seed(5)
    x = torch.zeros((m, d), dtype=torch.bfloat16, device=DEV)
    x[:, :2] = 256.0
    x[:, 127] = 448.0                                         # the row's scale is 1
    differ = 0
    for factor in (1.0 + torch.rand(12, generator=gen)).tolist():
        factor = torch.tensor(factor, device=DEV)
        w_in, w_out = _feed_forward(d, factor)
        up = torch.zeros(128, device=DEV)
        up[:80] = factor * torch.tensor([v + h for v, h in _middles()], device=DEV)
        up[80] = factor * 448.0
        h = up * 2.0 ** 13
        s = h[80] / torch.tensor(448.0, device=DEV)
        q = (h / s).to(torch.float8_e4m3fn).float()
        differ += int((q != (h * (1.0 / s)).to(torch.float8_e4m3fn).float()).sum())
        got = ops.glu_mlp_fp8(x, w_in, w_out)
        assert torch.equal(got, (q * s).to(torch.bfloat16).expand(m, 128))
    assert differ > 50                                        # (the middles do tell the two apart)
    ops.check_tcgen05_errors(torch.device(DEV))


@pytest.mark.parametrize("exponent", [-149, -140, -127, -126, -120, -100, -90, -81, -80, -79, -64, 0, 63, 90, 98, 99, 100, 101, 110, 119])
def test_rows_of_any_size_are_quotients(exponent):
    """rows whose largest numbers are a few hundred 2^exponent (as far as fp32 has them), the others down to nought: the numbers of torch's own division"""
    from mimirmind_b200.kernels import ops
    gen = torch.Generator(device=DEV).manual_seed(exponent + 200)
    x = torch.randn((64, 640), generator=gen, device=DEV, dtype=torch.float64) * torch.exp2(-12.0 * torch.rand((64, 640), generator=gen, device=DEV, dtype=torch.float64))
    x = (100.0 * x * 2.0 ** exponent).float()
    assert bool(x.isfinite().all()) and bool((x != 0).any())
    s = (x.view(64, 5, 128).abs().amax(dim=2) / torch.full((64, 5), 448.0, device=DEV)).clamp_min(2.0 ** -126)
    q = (x.view(64, 5, 128) / s.unsqueeze(2)).to(torch.float8_e4m3fn).view(64, 640)
    got = ops.quantize_fp8_rows(x)
    assert torch.equal(got.scales, s) and torch.equal(got.values.float(), q.float())
