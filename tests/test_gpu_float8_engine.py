"""Engines whose layers keep their matrices in 8 bits, on the GPU: against the same engine over 64-bit kernels on the CPU, in every cut of the
work, and through every architecture that has such parts."""

import importlib

import numpy as np
import pytest
import torch

import beholdd
from float8_emulation import Float8TorchKernels
from test_float8_engine import QWEN

pytestmark = pytest.mark.gpu

# A value next to a border between two e4m3 numbers falls on its other side where sums differ by their rounding: 2^-3 of the value at most, for
# at most one value in a thousand where sums are float32 (2^-24 of sums of some hundred terms, borders 2^-4 of a value apart), so sqrt(1e-3) / 8 =
# 0.4 % of a product's input by norm, and 4 products a layer of two: 1.2 %.  bfloat16 activations alone are 2^-9 off in each of about ten
# roundings a layer, and a value in sixteen lies within that of a border: sqrt(1/16) / 8 = 3.2 % a product by norm, 9 % for eight.
NORM = {"float32": 0.012, "bfloat16": 0.09}


def _off(got, want):
    got, want = got.float().cpu(), want.float()
    return float((got - want).norm() / want.norm())


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    path = str(tmp_path_factory.mktemp("float8"))
    beholdd.write_random_model(path, QWEN, seed=3, dtype="float32", std=0.08)
    return path


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_every_cut_of_the_work(folder, dtype):
    """Whole prompts, portions, single tokens through captured steps, and a batch: as the CPU's engine, and as each other."""
    engine = beholdd.Engine(folder, dtype=dtype, max_tokens=2048, device="cuda:0", weights="float8")
    double = beholdd.Engine(folder, dtype=dtype, max_tokens=2048, device="cpu", kernels=Float8TorchKernels(), weights="float8")
    rng = np.random.default_rng(4)
    prompt = [int(t) for t in rng.integers(0, 384, size=150)]
    everywhere = list(range(150))
    want = double.step([beholdd.StepEntry(double.alloc_slot(), prompt, everywhere)])
    whole = engine.step([beholdd.StepEntry(engine.alloc_slot(), prompt, everywhere)]).clone()
    assert _off(whole, want) < NORM[dtype]
    slot, rows = engine.alloc_slot(), []
    for first, last in ((0, 20), (20, 60), (60, 100), (100, 130)):
        rows.append(engine.step([beholdd.StepEntry(slot, prompt[first:last], list(range(last - first)))]).clone())
    for at in range(130, 150):
        rows.append(engine.step([beholdd.StepEntry(slot, [prompt[at]], [0])]).clone())
    assert _off(torch.cat(rows), want) < NORM[dtype]
    others = [engine.alloc_slot() for _ in range(3)]
    batch = engine.step([beholdd.StepEntry(s, prompt[:n], [n - 1]) for s, n in zip(others, (7, 40, 90))])
    assert _off(batch, want[[6, 39, 89]]) < 2 * NORM[dtype]      # (three rows rather than 150: their norm varies more)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("batch", [20, 60, 130])
def test_captured_steps_of_many_sequences(folder, dtype, batch):
    """Every replay of a step whose norms write rows in 8 bits, with eager steps between, as the CPU's engine has the same positions."""
    engine = beholdd.Engine(folder, dtype=dtype, max_tokens=(batch + 1) * 64, max_slots=batch + 1, device="cuda:0", weights="float8")
    double = beholdd.Engine(folder, dtype=dtype, max_tokens=512, device="cpu", kernels=Float8TorchKernels(), weights="float8")
    prompt = [int(t) for t in np.random.default_rng(8).integers(0, 384, size=40)]
    want = double.step([beholdd.StepEntry(double.alloc_slot(), prompt, list(range(40)))])
    slots, lengths = [engine.alloc_slot() for _ in range(batch)], [5 + i % 25 for i in range(batch)]
    engine.step([beholdd.StepEntry(slot, prompt[:n], [n - 1]) for slot, n in zip(slots, lengths)])
    for t in range(6):
        got = engine.step([beholdd.StepEntry(slot, [prompt[n + t]], [0]) for slot, n in zip(slots, lengths)]).clone()
        assert _off(got, want[[n + t for n in lengths]]) < 2 * NORM[dtype], f"step {t}"
        other = engine.alloc_slot()
        engine.step([beholdd.StepEntry(other, prompt[:30], [29])])
        engine.free_slot(other)
        torch.cuda.synchronize()


def test_generation_in_8_bits(folder):
    """Greedy tokens of the loop that runs ahead are those of its own steps one by one."""
    engine = beholdd.Engine(folder, dtype="bfloat16", max_tokens=1024, device="cuda:0", weights="float8")
    prompts = [[5, 17, 3], [9], list(range(40))]
    results = engine.generate(prompts, max_new_tokens=12)
    for prompt, result in zip(prompts, results):
        slot = engine.alloc_slot()
        assert len(result.token_ids) == 12
        fed = list(prompt)
        logits = engine.step([beholdd.StepEntry(slot, fed, [len(fed) - 1])])
        for token in result.token_ids:
            row = logits[0].float().cpu()
            assert row[token] >= row.max() - NORM["bfloat16"] * row.abs().max()
            logits = engine.step([beholdd.StepEntry(slot, [token], [0])])
        engine.free_slot(slot)
    assert engine.memory_plan()


MODELS = [("gokazen", "mixed"), ("pudorax", "mixed"), ("dupidra", "mixed"), ("vepelix", "mixed"), ("lurepel", "mixed"), ("vitudra", "mixed")]


@pytest.mark.parametrize("name,which", MODELS)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_every_architecture(name, which, dtype, tmp_path):
    """A prompt and single tokens behind it: finite logits, the layers' matrices in 8 bits, and in a float32 engine the median position as over 64-bit
    kernels (a choice of experts next to a border may go another way, and a position with it)."""
    from beholdd.kernels.library import Float8Weight
    models = importlib.import_module(f"{name}_models")
    config = models.CONFIGS[which]
    models.write_model(str(tmp_path), config, models.random_weights(config, seed=5))
    engine = beholdd.Engine(str(tmp_path), dtype=dtype, max_tokens=1024, device="cuda:0", weights="float8")
    found, stack, seen = 0, list(engine.model.own_blocks()), set()
    while stack:
        thing = stack.pop()
        if id(thing) in seen:
            continue
        seen.add(id(thing))
        if isinstance(thing, Float8Weight):
            found += 1
        elif isinstance(thing, (list, tuple)):
            stack += thing
        elif isinstance(thing, dict):
            stack += thing.values()
        elif hasattr(thing, "__dict__") and not isinstance(thing, type):
            stack += vars(thing).values()
    assert found >= 2 * len(list(engine.model.own_blocks()))
    vocab = engine.model.vocab
    rng = np.random.default_rng(6)
    tokens = [int(t) for t in rng.integers(0, vocab, size=48)]
    slot = engine.alloc_slot()
    rows = [engine.step([beholdd.StepEntry(slot, tokens[:40], list(range(40)))]).float().cpu()]
    for token in tokens[40:]:
        rows.append(engine.step([beholdd.StepEntry(slot, [token], [0])]).float().cpu())
    got = torch.cat(rows)
    assert bool(torch.isfinite(got).all())
    if dtype == "float32":
        double = beholdd.Engine(str(tmp_path), dtype=dtype, max_tokens=1024, device="cpu", kernels=Float8TorchKernels(), weights="float8")
        want = double.step([beholdd.StepEntry(double.alloc_slot(), tokens, list(range(48)))])
        off = (got - want).norm(dim=1) / want.norm(dim=1)
        assert float(off.median()) < 0.05


def test_the_byte_plan_bounds_what_is_allocated(tmp_path):
    """Wide enough that matrices, not the allocator's units, are the bytes."""
    config = dict(QWEN, hidden_size=1024, intermediate_size=2816, num_attention_heads=8, head_dim=128, num_hidden_layers=3, max_position_embeddings=1024)
    beholdd.write_random_model(str(tmp_path), config, seed=1)
    kept = {}
    for weights in ("stored", "float8"):
        torch.cuda.empty_cache()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        engine = beholdd.Engine(str(tmp_path), dtype="bfloat16", max_tokens=1024, max_slots=4, device="cuda:0", weights=weights, max_rows_per_step=512)
        kept[weights] = torch.cuda.memory_allocated() - before
        slot = engine.alloc_slot()
        engine.step([beholdd.StepEntry(slot, [3] * 500, [499])])
        for _ in range(3):
            engine.step([beholdd.StepEntry(slot, [7], [0])])
        torch.cuda.synchronize()
        assert torch.cuda.max_memory_allocated() - before <= engine.plan.total_bytes
        del engine
    assert kept["float8"] < 0.75 * kept["stored"]
