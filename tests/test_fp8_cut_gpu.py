"""What a token of a routed-experts layer in 8 bits is multiplied with, by how many tokens share its step: up to 16 keep their rows' bits, from 17 on rows and hidden rows are e4m3."""
import pytest
import torch

import fp8_util as f8
import test_fp8_engine_gpu as base

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _part(d, f, experts, top, gen):
    from mimirmind_b200.config.spec import PartSpec
    from mimirmind_b200.parts.base import WeightView
    from mimirmind_b200.registry import FEED_FORWARDS
    rnd = lambda *s: (0.1 * torch.randn(s, generator=gen, device=DEV)).to(torch.bfloat16)     # noqa: E731
    w = {"r": 0.3 * torch.randn((experts, d), generator=gen, device=DEV),
         **{f"e{e}.{k}": rnd(*((d, f) if k == "down" else (f, d))) for e in range(experts) for k in ("gate", "up", "down")}}
    spec = {"hidden": d, "ff": f, "experts": experts, "top": top, "router": "r", "expert": "e{}"}
    return FEED_FORWARDS.get("routed_experts")(PartSpec("routed_experts", spec), WeightView(w), base._rt())


def _e4m3_off(v, err=0.0):
    """The most that quantising rows that may be off by ``err`` changes their numbers: half a step of e4m3 is 2^-4 of a number, and 2^-10 of the scale below 2^-6
    of it; the scale is the block's largest number / 448, its rounding 2^-24"""
    m, k = v.shape
    size = torch.nn.functional.pad(v.abs() + err, (0, -k % 128)).view(m, -1, 128)
    scale = size.amax(dim=2, keepdim=True) / 448.0
    return ((size * (2.0 ** -4 + 2.0 ** -20) + scale * 2.0 ** -10).view(m, -1))[:, :k]


@pytest.mark.parametrize("d,f,experts,top", [(128, 72, 6, 2), (272, 128, 16, 4)])
def test_a_token_among_sixteen_and_among_seventeen(d, f, experts, top):
    """the two results differ by no more than quantising the rows and the hidden rows can change them"""
    from mimirmind_b200.kernels import ops
    gen = base._gen(d, f, experts)
    part = _part(d, f, experts, top, gen)
    x = torch.randn((17, d), generator=gen, device=DEV).to(torch.bfloat16)
    few, many = part.forward(x[:16], None).double(), part.forward(x, None)[:16].double()
    idx, wts = ops.moe_router(x, part.w_router, top, 1, 1)
    w_in, w_out = base._wide(part.w_in), base._wide(part.w_out)
    most = torch.zeros((16, d), dtype=torch.float64, device=DEV)
    for t in range(16):
        row = x[t:t + 1].double()
        for c in range(top):
            e, weight = int(idx[t, c]), wts[t, c].double()
            (g, ge), (u, ue) = f8.product(row, w_in[e][0], off=_e4m3_off(row)), f8.product(row, w_in[e][1], off=_e4m3_off(row))
            h = f8.act64(g, u, "silu", 0.0)
            he = 1.1 * ge * (u.abs() + ue) + g.abs() * ue + h.abs() * 2.0 ** -11      # silu' is below 1.1, |silu(g)| below |g|
            y, ye = f8.product(h, w_out[e], off=he + _e4m3_off(h, he))
            most[t] += (weight * ye + weight * y.abs() * 2.0 ** -17)[0]
    tolerance = most + (few.abs() + many.abs()) * 2.0 ** -8                           # both are rounded to bf16
    assert bool(((few - many).abs() <= tolerance).all())
    off = float((few - many).norm() / few.norm())
    assert 0.0 < off < 0.1, off            # (half a step is at most 1 / 16 of a number; three roundings in a row of random signs stay well below 2^-4 sqrt(3) = 0.108)
    # among as many as take one path a token's bits do not depend on how many
    assert torch.equal(part.forward(x[:3], None), part.forward(x[:16], None)[:3])
    assert torch.equal(part.forward(torch.cat([x, x, x]), None)[:17], part.forward(x, None))
