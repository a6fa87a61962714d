"""What engines with 8-bit weights plan to allocate, without a GPU."""

import math
import random

import pytest

from beholdd.engine.memory import step_size
from beholdd.kernels.library import Float8Rows, KernelSizes
from beholdd.parts.experts import RoutedExperts


@pytest.fixture(scope="module")
def sizes():
    return KernelSizes(verbose_build=False)


def _unit(n_bytes):
    return -(-n_bytes // 512) * 512


def _experts_allocate(lib, n, top, experts, width, ff):
    """The tensors of one call of `experts_float8`, as it makes them."""
    pairs = n * top
    if lib.bh_experts_float8_one(pairs, top):
        return _unit(4 * pairs * ff)
    results = _unit(4 * pairs * width)
    if lib.bh_experts_float8_few(pairs, experts):
        return results + _unit(4 * pairs * ff)
    return (results + _unit(4 * experts * pairs) + _unit(4 * experts) + sum(map(_unit, Float8Rows.bytes_of(n, width))) + sum(map(_unit, Float8Rows.bytes_of(pairs, ff))))


def _experts_cases():
    rng = random.Random(3)
    between = lambda low, high: round(math.exp(rng.uniform(math.log(low), math.log(high))))
    yield 4096, 8, 32, 64, 8
    for _ in range(200):
        yield between(1, 5000), rng.randint(1, 12), between(1, 200), between(1, 3000), between(1, 2000)


def test_experts_plan_what_they_allocate(sizes):
    """For the planned number of rows and for fewer, narrow experts among them, whose rows in 8 bits have whole stretches."""
    for n, top, experts, width, ff in _experts_cases():
        planned = sizes.experts_float8_working_bytes(n, top, experts, width, ff)
        for rows in sorted({1, min(2, n), n // 3 + 1, max(n - 1, 1), n, *(min(max(count // top, 1), n) for count in (32, 128, 1000, 1024, 1030, 8 * experts, 8 * experts + top))}):
            assert _experts_allocate(sizes.lib, rows, top, experts, width, ff) <= planned, (rows, n, top, experts, width, ff)


@pytest.mark.parametrize("rows", [1, 300, 4096])
def test_the_part_plans_its_experts(sizes, rows):
    part = RoutedExperts(64, 32, 8, 8, float("inf"), "m.", router_bias=False)
    part.keep_in_float8()
    step = step_size(type("Model", (), {}), rows, 1, 2, 8192, sizes)
    # the router's logits (kept 128 wide where the rows are many), the choices and their weights, the input in another form
    beside = _unit(4 * rows * (128 if rows > 32 else 32)) + 2 * _unit(4 * rows * 8) + _unit(2 * rows * 64)
    assert part.working_bytes(step) >= _experts_allocate(sizes.lib, rows, 8, 32, 64, 8) + beside


# ---- weights ---------------------------------------------------------------------------------------------------------

WIDE = {"architectures": ["Qwen3ForCausalLM"], "num_hidden_layers": 12, "hidden_size": 512, "num_attention_heads": 8, "num_key_value_heads": 2,
        "head_dim": 64, "intermediate_size": 1408, "vocab_size": 384, "rope_theta": 1000000.0, "rms_norm_eps": 1e-5, "max_position_embeddings": 512,
        "tie_word_embeddings": False}


def experts_config():
    """Layers of 24 experts and one shared, most of the model's bytes."""
    import vepelix_models as models
    moe = lambda: models.moe(24, 2, 256, shared=256)
    return {"architecture": "Vepelix", "vocab": 211, "width": 512, "norm": {"eps": 1e-6},
            "layers": [models.latent(8, 32, 32, 32, 96, 96, 0.15, mlp=moe()), models.latent(8, 32, 32, 32, 96, 96, 0.15, mlp=moe()),
                       models.latent(8, 32, 32, 32, 96, 96, 0.15, mlp=moe())]}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    import beholdd
    import vepelix_models as models
    dense, experts = (str(tmp_path_factory.mktemp(name)) for name in ("dense", "experts"))
    beholdd.write_random_model(dense, WIDE, seed=1, dtype="bfloat16", std=0.05)
    models.write_model(experts, experts_config(), models.random_weights(experts_config(), seed=1))
    return {"dense": dense, "experts": experts}


def _plan(folder, weights, sizes, dtype="bfloat16"):
    """(the plan of an engine of that folder, as the engine and --plan-only make it; the model)."""
    from beholdd.cache import SequenceCache
    from beholdd.engine.engine import open_model, parse_dtype
    from beholdd.engine.memory import loaded_bytes, plan_memory
    act_size = {"bfloat16": 2, "float32": 4}[dtype]
    model, bound = open_model(folder, dtype, "cpu", weights)
    try:
        cache = SequenceCache(model.entry_needs, 256, parse_dtype(dtype), "cpu", sizes.PAGE, max_slots=2, max_position=model.max_position)
        return plan_memory(model, loaded_bytes(model, bound, sizes), cache.plan(), act_size, sizes, 64, 2, cache.max_position, sizes.PAGE, 4, weights=bound), model
    finally:
        bound.reader.close()


@pytest.mark.parametrize("which", ["dense", "experts"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_the_plan_shows_what_8_bits_save(folders, sizes, which, dtype):
    """One layer as it is stored, all layers in a byte a value, and nothing more; most of the bytes of these models are their layers' matrices."""
    from beholdd.engine.memory import _in_float8
    stored, _ = _plan(folders[which], "stored", sizes, dtype)
    plan, model = _plan(folders[which], "float8", sizes, dtype)
    act_size = {"bfloat16": 2, "float32": 4}[dtype]
    layers = [sum(matrices * rows * cols for _, matrices, rows, cols, _ in _in_float8(block)) for block in model.own_blocks()]
    assert min(layers) > 1e6
    beside = max(max(act_size * apart * rows * cols, sizes.float8_packing_bytes(rows, cols)) for block in model.own_blocks() for _, _, rows, cols, apart in _in_float8(block))
    saved = (act_size - 1.05) * sum(layers) - act_size * max(layers) - beside      # (scales and whole blocks are 5 %)
    assert saved > 0 and plan.total_bytes < stored.total_bytes - saved
    assert plan.total_bytes > sum(layers) + act_size * max(layers)


def test_a_layer_as_it_is_stored_is_planned_in_its_files_type(tmp_path, sizes):
    """A float32 tensor is read as float32 by a bfloat16 engine too."""
    import beholdd
    plans = {}
    for dtype in ("bfloat16", "float32"):
        beholdd.write_random_model(str(tmp_path / dtype), WIDE, seed=1, dtype=dtype, std=0.05)
        plans[dtype] = _plan(str(tmp_path / dtype), "float8", sizes)[0]
    label = "largest transient while the weights are loaded and regrouped"
    assert plans["float32"].bytes_of(label) >= plans["bfloat16"].bytes_of(label) + 2 * (512 * 768 + 512 * 512 + 3 * 512 * 1408)


def test_a_limit_that_stored_weights_exceed_lets_8_bits_through(folders, sizes):
    import io

    import beholdd
    stored, plan = _plan(folders["dense"], "stored", sizes)[0].total_bytes, _plan(folders["dense"], "float8", sizes)[0].total_bytes
    for weights, fits in (("stored", False), ("float8", True)):
        status = beholdd.cli.main(["generate", "--model", folders["dense"], "--weights", weights, "--plan-only", "--prompt-ids", "1,2", "--max-tokens", "256", "--slots", "2",
                                   "--max-rows-per-step", "64", "--memory-budget-bytes", str((stored + plan) // 2)], out=io.StringIO())
        assert (status == 0) == fits


@pytest.mark.parametrize("which", ["dense", "experts"])
def test_layers_are_brought_into_8_bits_in_turn(folders, which, monkeypatch):
    """No tensor of a layer is read while a matrix of another layer still stands as it is stored."""
    import torch

    import beholdd
    from beholdd.engine import engine as engine_module
    from beholdd.weights.binder import BoundWeights
    from float8_emulation import Float8TorchKernels

    opened = []
    real_open, real_get = engine_module.open_model, BoundWeights.__call__
    monkeypatch.setattr(engine_module, "open_model", lambda *args: opened.append(real_open(*args)) or opened[-1])

    def stored_layers(model):
        found = set()
        for index, block in enumerate(model.own_blocks()):
            feed_forward = block.feed_forward
            linears = [block.mixer.out, *(getattr(feed_forward, name) for name in ("gate_up", "down") if hasattr(feed_forward, name))]
            if any(isinstance(linear.weight, torch.Tensor) for linear in linears) or getattr(feed_forward, "w_down", None) is not None:
                found.add(index)
        return found

    held = []

    def get(self, name):
        if opened:
            held.append((name, stored_layers(opened[-1][0])))
        return real_get(self, name)

    monkeypatch.setattr(BoundWeights, "__call__", get)
    engine = beholdd.Engine(folders[which], dtype="float32", max_tokens=64, device="cpu", kernels=Float8TorchKernels(), weights="float8")
    assert not stored_layers(engine.model) and max(len(layers) for _, layers in held) <= 1
    assert len({name for name, _ in held}) > 30
    assert bool(torch.isfinite(engine.step([beholdd.StepEntry(engine.alloc_slot(), [3, 4, 5], [2])])).all())
