"""A model whose products hold their weights in 4 bits holds them in no other form."""

import gc
import weakref

import pytest
import torch

from thing_htn_2026_b200 import ops
from thing_htn_2026_b200.config import config_from_dict, named_config_json
from thing_htn_2026_b200.models.decoder import tensor_specs_of_plan
from thing_htn_2026_b200.parts import Runtime, block, part_class
from thing_htn_2026_b200.weights.random_init import random_tensors_on_device

DESIGNS = ["tiny-a", "lanilix-tiny", "bunudra-tiny", "ditilix-tiny", "dubazen-tiny", "futepel-tiny", "turutar-tiny"]


def layers_of(name):
    """The design's layers on the CPU, and nothing else that holds their tensors."""
    plan = config_from_dict(named_config_json(name)).plan()
    tensors = random_tensors_on_device(tensor_specs_of_plan(plan), 0, torch.bfloat16, torch.device("cpu"), 0.02, 0.02)
    runtime = Runtime(torch.bfloat16, torch.device("cpu"), tensors)
    layers = [part_class("block", layer.block.kind)(layer.block, runtime) for layer in plan.layers]
    runtime.tensors = {}
    return layers


def storages(thing, seen, found):
    """The storages of the tensors that hang on a part."""
    if id(thing) in seen:
        return
    seen.add(id(thing))
    if isinstance(thing, torch.Tensor):
        found[thing.untyped_storage().data_ptr()] = thing.untyped_storage().nbytes()
    elif isinstance(thing, dict):
        for v in thing.values():
            storages(v, seen, found)
    elif isinstance(thing, (list, tuple)):
        for v in thing:
            storages(v, seen, found)
    elif hasattr(thing, "__dict__"):
        storages(vars(thing), seen, found)


@pytest.mark.parametrize("name", DESIGNS)
def test_nothing_keeps_the_weights_that_were_replaced(name, monkeypatch):
    monkeypatch.setattr(block, "PARALLEL_STREAMS", False)
    monkeypatch.setattr(ops, "quantize_mx4", lambda w: ops.Mx4.__new__(ops.Mx4)._set(torch.empty(0, dtype=torch.uint8), *w.shape))
    layers = layers_of(name)
    held = [w for layer in layers for _, _, w in layer.products()]
    assert len(held) >= len(layers) and all(isinstance(w, torch.Tensor) for w in held)
    gone = {w.untyped_storage().data_ptr(): w.untyped_storage().nbytes() for w in held}
    alive = [weakref.ref(w) for w in held]
    before = {}
    storages(layers, set(), before)
    assert all(layer.quantize_products() for layer in layers)
    del held
    gc.collect()
    after = {}
    storages(layers, set(), after)
    assert not [ref for ref in alive if ref() is not None]
    assert sum(after.values()) == sum(before.values()) - sum(gone.values())
    # and no other tensor of a layer is as large as a weight that went: none was a copy of one
    wide = ("w_wide", "table", "w_up", "w_gate_up", "w_down")          # documented: they stay in 16 bits
    kept = [t for layer in layers for part in [layer] + layer.parts() for n, t in vars(part).items() if n not in wide and isinstance(t, torch.Tensor)]
    assert sum(t.numel() * t.element_size() for t in kept) < sum(gone.values()) / 4


def test_one_weight_at_a_time_is_held_in_both_forms(monkeypatch):
    monkeypatch.setattr(block, "PARALLEL_STREAMS", False)
    gone = []

    def quantize(w):
        assert all(ref() is None for ref in gone)
        gone.append(weakref.ref(w))
        return ops.Mx4.__new__(ops.Mx4)._set(torch.empty(0, dtype=torch.uint8), *w.shape)

    monkeypatch.setattr(ops, "quantize_mx4", quantize)
    for layer in layers_of("tiny-a"):
        layer.quantize_products()
    assert len(gone) > 4


@pytest.mark.parametrize("name", DESIGNS)
def test_a_weight_is_held_once(name, monkeypatch):
    """In 16 bits, too: a mixer pair's members do not keep what the pair's products have copies of."""
    monkeypatch.setattr(block, "PARALLEL_STREAMS", False)
    config = config_from_dict(named_config_json(name))
    layers, found = layers_of(name), {}
    storages(layers, set(), found)
    plan = config.plan()
    specs = {s.name: s for layer in plan.layers for s in part_class("block", layer.block.kind).tensor_specs(layer.block)}
    shapes = random_tensors_on_device(list(specs.values()), 0, torch.bfloat16, torch.device("cpu"), 0.02, 0.02)
    wanted = sum(t.numel() * 2 for t in shapes.values() if t.dim() > 1)
    assert sum(found.values()) <= 1.25 * wanted


@pytest.mark.gpu
@pytest.mark.parametrize("name", DESIGNS)
def test_bytes_of_a_model_on_the_device(name):
    from thing_htn_2026_b200.engine.loading import random_model
    model = random_model(config_from_dict(named_config_json(name)), 5, "bfloat16", "cuda:0")
    gc.collect()
    products = [w for layer in model.layers for _, _, w in layer.products()]
    piece = 512                                                # what the allocator rounds to
    gone = {w.untyped_storage().data_ptr(): -(-w.untyped_storage().nbytes() // piece) * piece for w in products}
    del products
    before = torch.cuda.memory_allocated()
    model.quantize("mx4")
    gc.collect()
    held = sum(-(-w.nbytes // piece) * piece for layer in model.layers for _, _, w in layer.products())
    assert torch.cuda.memory_allocated() <= before - sum(gone.values()) + held


# What stays in 16 bits, as :meth:`DecoderModel.quantize` says.
STAYS = {"routers and routed experts": {"w_route", "w_up", "w_gate_up", "w_down"},
         "decays, step sizes, input and forget gates": {"w_a1", "w_a2", "w_gates", "w_bc", "w_dt", "w_low", "w1", "w2"},
         "time mixing's input projections": {"w_wide"}, "token rows": {"table", "w_gate", "w_proj"}}
EXPERTS = {"RoutedExperts", "RoutedGLUExperts", "RoutedClampedExperts"}


@pytest.mark.parametrize("name", DESIGNS)
def test_what_stays_in_16_bits(name, monkeypatch):
    monkeypatch.setattr(block, "PARALLEL_STREAMS", False)
    for layer in layers_of(name):
        for part in [layer] + layer.parts():
            products = getattr(part, "PRODUCTS", ())
            stays = {n for n, t in vars(part).items() if isinstance(t, torch.Tensor) and t.dim() > 1 and t.dtype == torch.bfloat16} - set(products)
            if type(part).__name__ in EXPERTS:
                assert stays and stays <= STAYS["routers and routed experts"]
            else:
                assert stays <= set.union(*STAYS.values()) - STAYS["routers and routed experts"], (type(part).__name__, stays)


def test_a_mixer_that_says_its_rows_itself():
    """A mixer in phases of a user's own: ``in_rows`` and ``out_rows`` of its own, and ``finish``."""
    from thing_htn_2026_b200.parts.fused import PhasedMixer

    class Own(PhasedMixer):
        def __init__(self):
            self.rows = [(torch.ones(8, 4), None), (torch.ones(4, 8), torch.zeros(4))]
            self.finish()

        def in_rows(self):
            return self.rows[0]

        def out_rows(self):
            return self.rows[1]

    own = Own()
    assert own.w_in is own.rows[0][0] and own.b_in is None and own.w_out is own.rows[1][0] and own.b_out is own.rows[1][1]
