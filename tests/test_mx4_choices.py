"""Formats that an engine does not take are refused before a model is loaded."""

import pytest

from thing_htn_2026_b200 import Engine, cli
from thing_htn_2026_b200.config import config_from_dict, named_config_json
from thing_htn_2026_b200.engine import engine as engine_module

BAD = [("int4", None), (None, "mx4"), ("mx4", "fp8"), ("mx4", ""), ("", None)]


@pytest.mark.parametrize("weights,activations", BAD)
def test_refused_ahead_of_the_load(weights, activations, monkeypatch):
    def loads(*args, **kwargs):
        raise AssertionError("a model was loaded")

    monkeypatch.setattr(engine_module, "load_model", loads)
    monkeypatch.setattr(engine_module, "random_model", loads)
    with pytest.raises(ValueError, match="mx4"):
        Engine("/no/such/folder", weights=weights, activations=activations)
    with pytest.raises(ValueError, match="mx4"):
        Engine.from_config(config_from_dict(named_config_json("tiny-a")), weights=weights, activations=activations)


def test_the_command_line_wants_weights_with_activations():
    with pytest.raises(SystemExit, match="--weights mx4"):
        cli.main(["generate", "--random-config", "tiny-a", "--prompt-lens", "5", "--max-new-tokens", "2", "--activations", "mx4"])
