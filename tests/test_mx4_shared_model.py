"""A model that several engines share: its weights are not replaced under one that computes with them, and each keeps its choice of rows."""

import gc

import pytest
import torch

from thing_htn_2026_b200 import Engine, ops
from thing_htn_2026_b200.config import config_from_dict, named_config_json
from thing_htn_2026_b200.engine.step import StepEntry
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


def test_which_rows_are_quantised(monkeypatch):
    monkeypatch.setattr(ops, "quantize_mx4", lambda x, to_multiply=False: "quantised")
    monkeypatch.setattr(ops, "linear_mx4", lambda x, *args: x)
    a, b = [ops.Mx4.__new__(ops.Mx4)._set(torch.zeros(ops._mx4_bytes(4, 64), dtype=torch.uint8), 4, 64, quantizes) for quantizes in (False, True)]
    x = torch.zeros(1, 64)

    def quantised():
        return [isinstance(ops.linear(x, w), str) for w in (a, b)]

    assert quantised() == [False, True]
    with ops.quantizing_rows_of(frozenset()):
        assert quantised() == [False, False]
        with ops.quantizing_rows_of(frozenset([a])):
            assert quantised() == [True, False]
        assert quantised() == [False, False]
    assert quantised() == [False, True]
    with pytest.raises(ZeroDivisionError):
        with ops.quantizing_rows_of(frozenset([a])):
            1 / 0
    assert quantised() == [False, True]


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


def logits_of(engine, prompts, n_steps):
    runner, cache = engine.backend.runner, engine.backend.cache
    slots = cache.open(len(prompts))
    with torch.inference_mode():
        out = [runner.step([StepEntry(s, p, (0, len(p) - 1)) for s, p in zip(slots, prompts)])]
        for i in range(n_steps):
            out.append(runner.step([StepEntry(s, [(7 * i + s) % 200], (0,)) for s in slots]))
    cache.close(slots)
    return torch.cat(out)


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [True, False])
def test_each_engine_keeps_its_choice_of_rows(graphs):
    prompts = [list(range(5, 12)), [3], list(range(40, 110))]
    alone = [engine_of("tiny-b", "bfloat16", weights="mx4", activations=activations) for activations in (None, "mx4")]
    want = [(logits_of(e, prompts, 2), list(e.generate(prompts, 9))) for e in alone]
    assert not torch.equal(want[0][0], want[1][0])
    first = engine_of("tiny-b", "bfloat16", weights="mx4", graphs=graphs)
    assert list(first.generate(prompts[:2], 4)) == list(alone[0].generate(prompts[:2], 4))       # graphs of two sequences
    engines = [first] + [Engine(None, dtype="bfloat16", model=first.model, max_tokens=1024, max_batch=4, graphs=graphs, weights="mx4", activations=a)
                         for a in ("mx4", None, "mx4")]
    engines.append(Engine(None, dtype="bfloat16", model=first.model, max_tokens=1024, max_batch=4, graphs=graphs))      # as the model is now
    late = Engine(None, dtype="bfloat16", model=first.model, max_batch=4, graphs=graphs, weights="mx4")                 # its cache comes with the first call
    first.model.quantize("mx4", "mx4")
    for _ in range(2):
        for engine, quantises in zip(engines, (0, 1, 0, 1, 1)):
            assert torch.equal(logits_of(engine, prompts, 2), want[quantises][0])
            assert list(engine.generate(prompts, 9)) == want[quantises][1]
        assert list(late.generate(prompts, 9)) == want[0][1]
