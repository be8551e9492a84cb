"""The memory that weights in 8 bits save is there for the cache."""
import pytest
import torch

pytestmark = pytest.mark.gpu
CONFIG = dict(architectures=["Qwen2ForCausalLM"], model_type="qwen2", vocab_size=512, hidden_size=1024, intermediate_size=16384, num_hidden_layers=6,
              num_attention_heads=8, num_key_value_heads=2, head_dim=128, rms_norm_eps=1e-6, rope_theta=1000000.0, max_position_embeddings=1 << 20, tie_word_embeddings=False)
MIB = 1 << 20


def _model(weights):
    from mimirmind_b200.engine.loader import random_model
    from mimirmind_b200.registry import _ensure_builtin, get_architecture
    _ensure_builtin()
    arch = get_architecture("Qwen2ForCausalLM")
    return random_model(arch.build_spec(arch.parse_config(CONFIG, "test")), 1, "bfloat16", weights=weights)


def _fits(model):
    """bytes of cache that the rule finds room for (no cap of contexts reached)"""
    from mimirmind_b200 import Engine
    from mimirmind_b200.cache import sizing
    tokens = Engine.cache_tokens_that_fit(model, 16, 1 << 20, 512, 1024, 0.9)
    assert tokens < (1 << 20) * 1024
    return tokens * sizing.cache_bytes_per_token(model.cache_groups(), 2)


def test_the_cache_is_sized_with_what_quantising_gave_back():
    """576 MiB of feed-forwards in bf16, given up for 288: whatever the allocator still holds of them, and of anything else that is given up, counts as room"""
    torch.cuda.empty_cache()
    model = _model("fp8")
    given_up = torch.empty(3000 * MIB, dtype=torch.uint8, device="cuda")
    del given_up
    found = _fits(model)
    torch.cuda.empty_cache()
    assert torch.cuda.memory_reserved() - torch.cuda.memory_allocated() < 128 * MIB
    assert abs(found - _fits(model)) < 64 * MIB


def test_a_model_is_quantised_as_it_is_loaded(tmp_path):
    """16 layers of 48 MiB of feed-forwards in bf16: at no time are all of them on the device"""
    from mimirmind_b200.engine.loader import load_model, random_model
    from mimirmind_b200.registry import _ensure_builtin, get_architecture
    from mimirmind_b200.weights import write_random_model
    _ensure_builtin()
    config = dict(CONFIG, intermediate_size=8192, num_hidden_layers=16)
    arch = get_architecture("Qwen2ForCausalLM")
    spec = arch.build_spec(arch.parse_config(config, "test"))
    write_random_model(str(tmp_path), config, 1, "bfloat16")
    for load in (lambda: random_model(spec, 1, "bfloat16", weights="fp8"), lambda: load_model(str(tmp_path), "bfloat16", weights="fp8")[0]):
        torch.cuda.empty_cache()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        model = load()
        assert torch.cuda.max_memory_allocated() - before < 16 * 48 * MIB
        del model
