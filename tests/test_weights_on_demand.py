"""Tensors that are read or made when a part asks for them."""
import pytest
import torch

from conftest import TINY
from mimirmind_b200.weights import load_spec, load_tensors, random_tensors, random_tensors_on_demand, tensors_on_demand, write_random_model
from mimirmind_b200.weights.store import TensorsOnDemand


def test_a_tensor_is_made_when_it_is_asked_for_and_not_kept_when_taken():
    made = []

    def make(name):
        made.append(name)
        return torch.full((2,), float(len(made)))

    t = TensorsOnDemand(["a", "b"], make)
    assert "a" in t and "c" not in t and not made
    assert t["a"] is t["a"] and made == ["a"]
    first = t["a"]
    assert t.pop("a") is first and made == ["a"] and "a" not in t
    assert t.pop("b").tolist() == [2.0, 2.0]
    for name in ("a", "b", "c"):
        with pytest.raises(KeyError):
            t.pop(name)
        with pytest.raises(KeyError):
            t[name]
    assert made == ["a", "b"]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_they_are_the_tensors_of_a_whole_load(tmp_path, dtype):
    folder = str(tmp_path)
    spec = write_random_model(folder, TINY["B"], 3, "bfloat16")
    _, spec = load_spec(folder)
    whole = load_tensors(folder, spec, dtype, "cpu")
    with tensors_on_demand(folder, spec, dtype, "cpu") as some:
        for name, t in whole.items():
            got = some.pop(name)
            assert got.dtype == t.dtype and torch.equal(got, t)
    at_once, later = random_tensors(spec, 7, dtype), random_tensors_on_demand(spec, 7, dtype)
    for name in reversed(list(at_once)):                    # in any order
        assert torch.equal(later[name], at_once[name])
