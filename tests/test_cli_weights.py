"""Modes that run with the weights as they are stored do not take another form in silence."""
import json

import pytest

from conftest import TINY
from mimirmind_b200 import cli


def test_modes_without_a_choice_of_weights_refuse_it(tmp_path):
    (tmp_path / "c.json").write_text(json.dumps(TINY["B"]))
    for args in (["replay", "--model", str(tmp_path), "--out", str(tmp_path), "--max-tokens", "64"],
                 ["random-weights", "--model-config", str(tmp_path / "c.json"), "--out", str(tmp_path / "m")]):
        with pytest.raises(SystemExit, match="--weights"):
            cli.main(args + ["--weights", "fp8"])
    assert not (tmp_path / "m").exists()
