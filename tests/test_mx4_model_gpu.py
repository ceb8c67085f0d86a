"""Models whose layers hold their weights in 4 bits, beside models whose layers hold what those weights stand for."""

import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import tiny
from plain import mx4_plain, qwen3_plain
from thing_htn_2026_b200 import Engine, ops
from thing_htn_2026_b200.config import config_from_dict, named_config_json
from thing_htn_2026_b200.engine.step import StepEntry
from thing_htn_2026_b200.weights import safetensors_io

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DESIGNS = ["tiny-a", "lanilix-tiny", "bunudra-tiny", "ditilix-tiny", "dubazen-tiny", "futepel-tiny", "turutar-tiny"]


def stand_for(w):
    return ops.dequantize_mx4(ops.quantize_mx4(w.contiguous()), w.dtype)


def engine_of(name, dtype, **kwargs):
    return Engine.from_config(config_from_dict(named_config_json(name)), seed=5, dtype=dtype, max_tokens=1024, max_batch=4, **kwargs)


def logits_of(engine, prompts, n_steps):
    """Float32 logits of the prompts' last places and of n_steps more tokens each, the same tokens whatever the model says."""
    runner, cache = engine.backend.runner, engine.backend.cache
    slots = cache.open(len(prompts))
    with torch.inference_mode():
        out = [runner.step([StepEntry(s, p, (0, len(p) - 1)) for s, p in zip(slots, prompts)])]
        for i in range(n_steps):
            out.append(runner.step([StepEntry(s, [(7 * i + s) % 200], (0,)) for s in slots]))
    cache.close(slots)
    return torch.cat(out)


def weights_as_values(engine):
    """The engine's layers multiply by what their weights would stand for in 4 bits; returns those weights."""
    kept = []
    for layer in engine.model.layers:
        for part in [layer] + layer.parts():
            for name in getattr(part, "PRODUCTS", ()):
                w = getattr(part, name)
                if isinstance(w, torch.Tensor):
                    setattr(part, name, stand_for(w))
                    kept.append(getattr(part, name))
    return kept


@pytest.mark.gpu
@pytest.mark.parametrize("activations", [None, "mx4"])
@pytest.mark.parametrize("name", DESIGNS)
def test_a_model_is_the_one_its_weights_stand_for(name, activations, monkeypatch):
    prompts = [list(range(3, 20)), [9], list(range(100, 170))]
    got = logits_of(engine_of(name, "float32", weights="mx4", activations=activations), prompts, 3)
    other = engine_of(name, "float32")
    kept = weights_as_values(other)
    assert len(kept) >= len(other.model.layers)
    if activations:
        ids, linear = {w.data_ptr() for w in kept}, ops.linear

        def with_rows(x, weight, *args, **kwargs):
            return linear(stand_for(x) if weight.data_ptr() in ids else x, weight, *args, **kwargs)

        monkeypatch.setattr(ops, "linear", with_rows)
    want = logits_of(other, prompts, 3)
    assert torch.isfinite(got).all()
    # Without quantised rows both differ by the order of float32 sums alone.  With them a difference of that size can carry an
    # entry over a midpoint, to the neighbouring magnitude: a quarter of it at most, in single entries.
    tolerance = 2e-2 if activations else 2e-4
    assert (got - want).abs().max() <= tolerance * want.abs().max(), (got - want).abs().max() / want.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["a", "b", "c"])
def test_logits_are_those_of_the_plain_model_with_these_values(name, tmp_path):
    """A folder whose projections are rounded to 4 bits by the definition, through the plain implementation."""
    folder, rounded = str(tmp_path / "model"), str(tmp_path / "rounded")
    tiny.write_model(folder, name)
    tensors = qwen3_plain.read_safetensors(os.path.join(folder, "model.safetensors"))
    for key, t in tensors.items():
        if key.endswith("_proj.weight"):
            values = mx4_plain.values(*mx4_plain.quantize(t.double().numpy()), t.shape[1])
            tensors[key] = torch.from_numpy(values).to(t.dtype)
    os.makedirs(rounded)
    safetensors_io.write_safetensors(os.path.join(rounded, "model.safetensors"), tensors)
    with open(os.path.join(folder, "config.json")) as src, open(os.path.join(rounded, "config.json"), "w") as dst:
        dst.write(src.read())
    engine = Engine(folder, dtype="float32", max_tokens=512, max_batch=2, weights="mx4")
    prompt = tiny.tokens(name, 37, 1)
    runner, cache = engine.backend.runner, engine.backend.cache
    (slot,) = cache.open(1)
    with torch.inference_mode():
        got = runner.step([StepEntry(slot, prompt, tuple(range(len(prompt))))]).cpu().numpy()
    want = qwen3_plain.model_logits(rounded, prompt).numpy()
    assert np.abs(got - want).max() <= 1e-4 * np.abs(want).max()


@pytest.mark.gpu
@pytest.mark.parametrize("activations", [None, "mx4"])
def test_generation_with_and_without_graphs_gives_the_same_tokens(activations):
    prompts = [list(range(5, 12)), [3], list(range(40, 110))]
    engines = [engine_of("tiny-b", "bfloat16", weights="mx4", activations=activations, graphs=g) for g in (True, False)]
    steps = [list(e.generate(prompts, 9, temperature=[0.0, 0.7, 0.0], seed=3)) for e in engines]
    assert steps[0] == steps[1] and len(steps[0]) == 9
    again = list(engines[0].generate(prompts, 9, temperature=[0.0, 0.7, 0.0], seed=3))
    assert again == steps[0]


@pytest.mark.gpu
def test_a_model_that_holds_4_bits_already_takes_the_choice_of_rows():
    first = engine_of("tiny-a", "float32", weights="mx4")
    held = [first.model.layers[0].mixer.w_qkv, first.model.layers[0].ffn.w_down]
    second = Engine(None, dtype="float32", model=first.model, max_tokens=1024, max_batch=4, weights="mx4", activations="mx4")
    assert second.model.layers[0].mixer.w_qkv is held[0] and all(w.quantizes_rows for w in held)


@pytest.mark.gpu
def test_from_the_command_line():
    done = subprocess.run([sys.executable, "-m", "thing_htn_2026_b200", "generate", "--random-config", "tiny-a", "--prompt-lens", "5,17",
                           "--max-new-tokens", "4", "--weights", "mx4", "--activations", "mx4"], cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stderr[-2000:]
    printed = [json.loads(line) for line in done.stdout.strip().splitlines()]
    engine = Engine.from_config(config_from_dict(named_config_json("tiny-a")), seed=0, weights="mx4", activations="mx4")
    from thing_htn_2026_b200 import cli
    steps = list(engine.generate(cli.make_prompts_of([5, 17], engine.model.vocab_size, 0), 4))
    assert [p["tokens"] for p in printed] == [[s[j] for s in steps] for j in range(2)]


def test_tensors_on_the_cpu_are_refused():
    with pytest.raises(ops.KernelError, match="CUDA only"):
        ops.quantize_mx4(torch.zeros(2, 64))
    with pytest.raises(ops.KernelError, match="CUDA only"):
        ops.mx4_from_parts(torch.zeros((2, 32), dtype=torch.uint8), torch.zeros((2, 2), dtype=torch.uint8), 64)
    with pytest.raises(ops.KernelError, match="CUDA only"):
        ops.Mx4(torch.zeros(768, dtype=torch.uint8), 4, 64)
    with pytest.raises(ops.KernelError, match="Mx4"):
        ops.linear_mx4(torch.zeros(2, 64), torch.zeros(3, 64))


def test_refused_choices():
    from thing_htn_2026_b200.models.decoder import DecoderModel
    model = DecoderModel.__new__(DecoderModel)
    model.layers = []
    model.quantize(None)
    for weights, activations in (("int4", None), (None, "mx4"), ("mx4", "fp8")):
        with pytest.raises(ValueError, match="mx4"):
            model.quantize(weights, activations)
    with pytest.raises(ValueError, match="no layer"):
        model.quantize("mx4")
