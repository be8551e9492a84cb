"""Every architecture with its feed-forwards and experts in 8 bits."""
import pytest
import torch

import bigerax_util
import domelix_util
import nefelorn_util
import segorax_util
import tupunex_util
import zubarax_util
from conftest import TINY

pytestmark = pytest.mark.gpu
CONFIGS = {f"{module.__name__[:-5]} {name}": cfg for module in (bigerax_util, domelix_util, nefelorn_util, segorax_util, tupunex_util, zubarax_util)
           for name, cfg in module.CONFIGS.items()} | {f"qwen2 {name}": cfg for name, cfg in TINY.items()}


@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_captured_steps_and_steps_one_by_one(name):
    """Prompts of several portions beside decoded tokens: a run gives the same tokens again, captured or not, the first step's logits are numbers and the same, and captured
    steps give what steps one by one give.  The last does not hold for Segorax in bf16, with stored weights either: the two cut latent attention's keys differently."""
    from mimirmind_b200 import Engine
    from mimirmind_b200.engine.loader import random_model
    from mimirmind_b200.engine.runner import StepEntry
    from mimirmind_b200.registry import _ensure_builtin, architecture_name, get_architecture
    from mimirmind_b200.weights import WeightsError
    _ensure_builtin()
    arch = get_architecture(architecture_name(CONFIGS[name]))
    spec = arch.build_spec(arch.parse_config(CONFIGS[name], "test"))
    prompts = [[(7 * i + 3 * s) % (spec.vocab_size - 1) for i in range(n)] for s, n in ((1, 5), (2, 110), (3, 33))]
    runs, logits = [], []
    for graphs in (True, True, False, False):
        try:
            model = random_model(spec, 5, "bfloat16", weights="fp8")
        except WeightsError:
            pytest.skip("a tensor's extent is only in a checkpoint")
        engine = Engine(model, cache_tokens=1024, max_context=240, token_budget=80, max_active=4, use_graphs=graphs)
        runs.append([r.tokens for r in engine.generate(prompts, max_new_tokens=20, use_eos=False)])
        assert engine.runner.add_request("a")
        logits.append(engine.runner.step([StepEntry("a", prompts[1][:70], [69])]).float())
    assert runs[0] == runs[1] and runs[2] == runs[3] and all(len(r) == 20 for r in runs[0] + runs[2])
    assert all(torch.equal(x, logits[0]) for x in logits) and bool(logits[0].isfinite().all())
    if not name.startswith("segorax"):
        assert runs[0] == runs[2]
