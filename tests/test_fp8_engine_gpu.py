"""Feed-forwards and experts in 8 bits as parts of a model, and whole models with them."""
import zlib

import pytest
import torch

import fp8_util as f8

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(*key):
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(repr(key).encode()))


def _rt():
    from mimirmind_b200.engine.loader import make_runtime
    return make_runtime(torch.bfloat16, weights="fp8")


def _wide(w):
    return w.values.float().double() * w.scales.double().repeat_interleave(128, -2)[..., :w.shape[-2], :].repeat_interleave(128, -1)[..., :w.shape[-1]]


def _close(got, y, err):
    tol = f8.rounded(y, err, got.dtype)
    off = (got.double() - y).abs()
    assert bool((off <= tol).all()), f"{(off - tol).max().item():.3g} over"


def _mlp64(x, part, act, limit):
    gate, up = _wide(part.w_in)
    h, err = f8.hidden64(f8.quantised(x)[0], gate, up, act, limit)
    h, off = f8.quantised(h, err)
    return f8.product(h, _wide(part.w_out), off=off)


@pytest.mark.parametrize("kind,act", [("swiglu", "silu"), ("swiglu", "gelu_tanh"), ("gated_mlp", "clamped")])
@pytest.mark.parametrize("m", [1, 9, 40, 300])
def test_feed_forward_parts(kind, act, m):
    from mimirmind_b200.config.spec import PartSpec
    from mimirmind_b200.parts.base import WeightView
    from mimirmind_b200.registry import FEED_FORWARDS
    gen = _gen(kind, act, m)
    d, f = 144, 200
    rnd = lambda *s: (0.1 * torch.randn(s, generator=gen, device=DEV)).to(torch.bfloat16)     # noqa: E731
    spec = PartSpec(kind, {"hidden": d, "intermediate": f, "gate": "g", "up": "u", "down": "d", "activation": act, "limit": 0.6})
    w = {"g": rnd(f, d), "u": rnd(f, d), "d": rnd(d, f)}
    kept = {k: v.clone() for k, v in w.items()}
    part = FEED_FORWARDS.get(kind)(spec, WeightView(w), _rt())
    assert part.native() is None and not w
    # a block's numbers are within half a step of its largest's: 2^-4 of a number, or half the smallest step
    for got, want in ((_wide(part.w_in)[0], kept["g"]), (_wide(part.w_in)[1], kept["u"]), (_wide(part.w_out), kept["d"])):
        assert ((got - want.double()).abs() <= want.double().abs() * 2.0 ** -4 + want.double().abs().max() * 2.0 ** -18).all()
    x = (20 * rnd(m, d)).contiguous()
    _close(part.forward(x, None), *_mlp64(x, part, act, 0.6))


@pytest.mark.parametrize("shared", [None, "plain", "gated"])
@pytest.mark.parametrize("n", [1, 16, 17, 150])
def test_routed_experts_part(n, shared):
    """few tokens, more tokens, a shared expert: the same sum as the operators on the part's own tensors"""
    from mimirmind_b200.config.spec import PartSpec
    from mimirmind_b200.kernels import ops
    from mimirmind_b200.parts.base import WeightView
    from mimirmind_b200.registry import FEED_FORWARDS
    gen = _gen(n, shared)
    d, f, experts, top = 128, 72, 6, 2
    rnd = lambda *s: (0.1 * torch.randn(s, generator=gen, device=DEV)).to(torch.bfloat16)     # noqa: E731
    params = {"hidden": d, "ff": f, "experts": experts, "top": top, "router": "r", "expert": "e{}"}
    w = {"r": 0.3 * torch.randn((experts, d), generator=gen, device=DEV), **{f"e{e}.{k}": rnd(*((d, f) if k == "down" else (f, d))) for e in range(experts) for k in ("gate", "up", "down")}}
    if shared:
        params["shared"] = PartSpec("swiglu", {"hidden": d, "intermediate": 96, "gate": "s.g", "up": "s.u", "down": "s.d"})
        w |= {"s.g": rnd(96, d), "s.u": rnd(96, d), "s.d": rnd(d, 96)}
        if shared == "gated":
            params["shared_gate"] = "sg"
            w["sg"] = rnd(1, d)
    part = FEED_FORWARDS.get("routed_experts")(PartSpec("routed_experts", params), WeightView(w), _rt())
    assert part.fp8 and not part.splits_weighed() and not w
    x = (10 * rnd(n, d)).contiguous()
    got = part.forward(x, None)
    idx, wts = ops.moe_router(x, part.w_router[:experts].contiguous(), top, 1, 1)
    routed = ops.moe_experts_fp8(x, idx, wts, part.w_in, part.w_out) if shared == "gated" or n > 16 else ops.moe_few(x, part.w_router, part.w_in, part.w_out, top)
    want = routed.double()
    if shared:
        gate = torch.sigmoid(x.double() @ part.w_router[experts:].double().t()) if shared == "gated" else 1.0
        want = want + gate * part.shared.forward(x, None).double()
    # one more rounding to bf16 (half a step: 2^-8), the gate in fp32
    assert ((got.double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -18) + 2.0 ** -20).all()
    branch = part.forward_split(x, None)
    assert branch.weights is None and branch.place is None and torch.equal(branch.rows, part._combined(x, None)[0]) and (branch.other is None) == (shared is None)


def _engine(name, weights, **kw):
    from mimirmind_b200 import Engine
    from mimirmind_b200.engine.loader import random_model
    from mimirmind_b200.registry import _ensure_builtin, architecture_name, get_architecture
    import domelix_util
    from conftest import TINY
    _ensure_builtin()
    cfg = domelix_util.CONFIGS["Q"] if name == "domelix" else TINY[name]
    arch = get_architecture(architecture_name(cfg))
    model = random_model(arch.build_spec(arch.parse_config(cfg, "test")), 5, "bfloat16", weights=weights)
    return Engine(model, cache_tokens=1024, max_context=400, token_budget=96, max_active=4, **kw)


@pytest.mark.parametrize("name", ["D", "E", "domelix"])
def test_models_run_with_weights_in_8_bits(name):
    """prompts of several portions beside decoded tokens: the captured decode steps give what steps one by one give, and the outputs stay near the
    stored weights' (the first step's logits: a rounding to e4m3 is off by half a step, 2^-4, at most, and only the feed-forwards are rounded)"""
    prompts = [[(7 * i + 3 * s) % 200 for i in range(n)] for s, n in ((1, 5), (2, 130), (3, 33))]
    runs = [_engine(name, "fp8", use_graphs=g).generate(prompts, max_new_tokens=20, use_eos=False) for g in (True, False)]
    for a, b in zip(*runs):
        assert a.tokens == b.tokens and len(a.tokens) == 20 and a.stats.finish_reason == b.stats.finish_reason
    from mimirmind_b200.engine.runner import StepEntry
    logits = []
    for weights in ("fp8", "stored"):
        eng = _engine(name, weights)
        assert eng.runner.add_request("a")
        logits.append(eng.runner.step([StepEntry("a", prompts[1][:90], [89])]).float())
    a, b = logits
    assert a.isfinite().all() and (a - b).norm() <= 0.25 * b.norm()


def test_weights_in_8_bits_are_refused_where_they_do_not_belong():
    from mimirmind_b200.engine.loader import make_runtime
    for kw in (dict(dtype="float32", weights="fp8"), dict(dtype="bfloat16", matmul="simt", weights="fp8"), dict(dtype="bfloat16", weights="int4")):
        with pytest.raises(ValueError):
            make_runtime(**kw)


def test_a_weight_filled_expert_by_expert_is_the_one_quantised_at_once():
    from mimirmind_b200.kernels import ops
    from mimirmind_b200.kernels.lib import KernelError
    w = 0.05 * torch.randn((5, 2, 140, 200), generator=_gen(1), device=DEV)
    whole, filled = ops.quantize_fp8_weight(w), ops.fp8_weight_like(5, 2, 140, 200, device=DEV)
    for e in range(5):
        ops.quantize_fp8_weight(w[e], out=filled, at=e)
    assert torch.equal(whole.scales, filled.scales) and torch.equal(whole.values.view(torch.uint8), filled.values.view(torch.uint8))
    for bad in (lambda: ops.quantize_fp8_weight(w[0], out=filled, at=5), lambda: ops.quantize_fp8_weight(w[0, 0], out=filled), lambda: ops.fp8_weight_like(3, device=DEV)):
        with pytest.raises(KernelError):
            bad()
