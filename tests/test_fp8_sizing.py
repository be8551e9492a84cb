"""What a step with weights in 8 bits needs beside the cache, counted before the cache is sized."""
from types import SimpleNamespace

import pytest

from mimirmind_b200.config.spec import PartSpec
from mimirmind_b200.kernels import lib, ops
from mimirmind_b200.parts.moe import fp8_step_bytes


def _spec(*layers):
    return SimpleNamespace(layers=[SimpleNamespace(feed_forward=p, extras=extras) for p, extras in layers])


def _mlp(d, f, kind="swiglu"):
    return PartSpec(kind, {"hidden": d, "intermediate": f})


def _experts(d, f, experts, top, **kw):
    return PartSpec("routed_experts", {"hidden": d, "ff": f, "experts": experts, "top": top, **kw})


def _rows(m, k):                # e4m3 rows from 16-byte boundaries and an fp32 scale per 128
    return m * (-(-k // 16) * 16) + 4 * m * -(-k // 128)


@pytest.mark.parametrize("n", [1, 16, 17, 520, 4104])
@pytest.mark.parametrize("d,f,experts,top", [(2048, 768, 128, 8), (4096, 64, 256, 1), (128, 1000, 4, 2), (100, 33, 6, 4)])
def test_the_experts_scratch_is_counted(n, d, f, experts, top):
    wanted = lib.load(verbose=False).mm_fp8_moe_experts_scratch(n, d, f, experts, top)
    assert wanted >= _rows(n, d) + _rows(n * top, d) + _rows(n * top, f) + 4 * n * top * d
    assert fp8_step_bytes(_spec((_experts(d, f, experts, top), {})), n) >= wanted
    # a shared expert's rows stand beside the routed ones' result
    for shared in (_mlp(d, 96), _mlp(d, 20 * d, "gated_mlp")):
        both = fp8_step_bytes(_spec((_experts(d, f, experts, top, shared=shared), {})), n)
        assert both >= wanted + _rows(n, d) + _rows(n, shared["intermediate"])


@pytest.mark.parametrize("n", [1, 300])
def test_feed_forwards_wherever_they_stand(n):
    wanted = _rows(n, 512) + _rows(n, 2000)
    assert fp8_step_bytes(_spec((_mlp(512, 2000), {})), n) >= wanted
    assert fp8_step_bytes(_spec((_mlp(64, 64), {}), (PartSpec("none"), {"second": _mlp(512, 2000, "gated_mlp"), "norm": PartSpec("rmsnorm", {"width": 512})})), n) >= wanted
    assert fp8_step_bytes(_spec((PartSpec("none"), {})), n) == 0
    # experts without gates keep the stored form; their shared expert does not
    assert fp8_step_bytes(_spec((_experts(64, 64, 4, 2, gated=False), {})), n) == 0
    assert fp8_step_bytes(_spec((_experts(64, 64, 4, 2, gated=False, shared=_mlp(512, 2000)), {})), n) >= wanted


def test_the_few_tokens_scratch_is_counted():
    d, f, top = 64, 4096, 32
    few = 16 * top * (4 * f + f // 2 + 24) + 32 + 36 * 16 * (d + 160)
    assert ops.moe_few_scratch(16, top, d, f) == few
    for n in (16, 40):
        assert fp8_step_bytes(_spec((_experts(d, f, 64, top), {})), n) >= few
