"""A model that several engines share: its weights are not replaced under one that computes with them."""

import gc

import pytest
import torch

from thing_htn_2026_b200 import Engine, ops
from thing_htn_2026_b200.config import config_from_dict, named_config_json
from thing_htn_2026_b200.models.decoder import DecoderModel
from thing_htn_2026_b200.parts.block import Block


class Layer(Block):
    PRODUCTS = ("w",)

    def __init__(self):
        self.w = torch.zeros(4, 64)


class User:
    pass


def bare_model():
    import weakref
    model = DecoderModel.__new__(DecoderModel)
    model.layers, model._users = [Layer()], weakref.WeakSet()
    return model


def test_weights_in_use_are_not_replaced(monkeypatch):
    monkeypatch.setattr(ops, "quantize_mx4", lambda w: ops.Mx4.__new__(ops.Mx4)._set(torch.zeros(ops._mx4_bytes(*w.shape), dtype=torch.uint8), *w.shape))
    model, user = bare_model(), User()
    held = model.layers[0].w
    model.used_by(user)
    for activations in (None, "mx4"):
        with pytest.raises(ValueError, match="computes with this model's weights"):
            model.quantize("mx4", activations)
        assert model.layers[0].w is held
    model.quantize(None)                      # nothing is changed
    del user
    gc.collect()
    model.quantize("mx4")
    quantized = model.layers[0].w
    assert isinstance(quantized, ops.Mx4)
    user = User()
    model.used_by(user)
    model.quantize("mx4")                     # nothing to replace
    assert model.layers[0].w is quantized


def engine_of(name, dtype, **kwargs):
    return Engine.from_config(config_from_dict(named_config_json(name)), seed=5, dtype=dtype, max_tokens=1024, max_batch=4, **kwargs)


@pytest.mark.gpu
@pytest.mark.parametrize("max_tokens", [None, 1024])
def test_an_engine_keeps_its_weights(max_tokens):
    """With its cache made ahead of the first call or by it."""
    prompts = [list(range(5, 12)), [3], list(range(40, 110))]
    first = Engine(None, dtype="bfloat16", model=engine_of("tiny-b", "bfloat16").model, max_tokens=max_tokens, max_batch=4)
    gc.collect()
    before = list(first.generate(prompts, 9)) if max_tokens else None
    weights = [w for layer in first.model.layers for _, _, w in layer.products()]
    with pytest.raises(ValueError, match="computes with this model's weights"):
        Engine(None, dtype="bfloat16", model=first.model, max_tokens=1024, max_batch=4, weights="mx4")
    with pytest.raises(ValueError, match="computes with this model's weights"):
        first.model.quantize("mx4")
    assert all(a is b for a, b in zip(weights, [w for layer in first.model.layers for _, _, w in layer.products()]))
    again = list(first.generate(prompts, 9))
    assert before is None or again == before
    plain = Engine(None, dtype="bfloat16", model=first.model, max_tokens=1024, max_batch=4)
    assert list(plain.generate(prompts, 9)) == again
    model = first.model
    del first, plain
    gc.collect()
    second = Engine(None, dtype="bfloat16", model=model, max_tokens=1024, max_batch=4, weights="mx4")
    fresh = engine_of("tiny-b", "bfloat16", weights="mx4")
    assert list(second.generate(prompts, 9)) == list(fresh.generate(prompts, 9))
