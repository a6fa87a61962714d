"""Engines whose layers keep their matrices in 8 bits: what is kept so, what is refused, and the router in groups as a part.  On the CPU."""

import io

import pytest
import torch

import beholdd
from beholdd.engine.engine import open_model
from beholdd.engine.memory import weights_as_kept
from beholdd.kernels.library import KernelSizes
from beholdd.parts.base import StepContext
from beholdd.parts.experts import RoutedExperts

import plain_float8 as plain
from float8_emulation import Float8Matrix, Float8TorchKernels
from kernel_emulation import TorchKernels

QWEN = {"architectures": ["Qwen3ForCausalLM"], "num_hidden_layers": 2, "hidden_size": 256, "num_attention_heads": 4, "num_key_value_heads": 2,
        "head_dim": 32, "intermediate_size": 320, "vocab_size": 384, "rope_theta": 1000000.0, "rms_norm_eps": 1e-5, "max_position_embeddings": 256,
        "tie_word_embeddings": False}


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    path = str(tmp_path_factory.mktemp("float8"))
    beholdd.write_random_model(path, QWEN, seed=3, dtype="float32", std=0.08)
    return path


def _engine(folder, **kw):
    kernels = Float8TorchKernels()
    return beholdd.Engine(folder, dtype="float32", max_tokens=256, device="cpu", kernels=kernels, weights="float8", **kw), kernels


def test_the_layers_matrices_are_kept_and_the_rest_is_not(folder):
    engine, kernels = _engine(folder)
    for block in engine.model.blocks:
        assert isinstance(block.mixer.qkv.weight, Float8Matrix) and isinstance(block.mixer.out.weight, Float8Matrix)
        assert block.feed_forward.gate_up.weight.matrices == 2 and isinstance(block.feed_forward.down.weight, Float8Matrix)
    assert isinstance(engine.model.head.linear.weight, torch.Tensor)
    engine.step([beholdd.StepEntry(engine.alloc_slot(), [5, 6, 7], [2])])
    assert kernels.products == 4 * len(engine.model.blocks)


def test_logits_are_the_stored_weights_up_to_the_roundings(folder):
    """Roundings of 2^-5 on average of every weight and activation leave logits a tenth off at most, and in the same order of size."""
    engine, _ = _engine(folder)
    stored = beholdd.Engine(folder, dtype="float32", max_tokens=256, device="cpu", kernels=TorchKernels())
    prompt = [3, 1, 4, 1, 5, 9, 2, 6]
    a = engine.step([beholdd.StepEntry(engine.alloc_slot(), prompt, list(range(8)))])
    b = stored.step([beholdd.StepEntry(stored.alloc_slot(), prompt, list(range(8)))])
    off = float((a - b).norm() / b.norm())
    assert 1e-4 < off < 0.15


def test_refusals(folder):
    with pytest.raises(ValueError, match="8 bits"):
        beholdd.Engine(folder, dtype="float32", max_tokens=64, device="cpu", kernels=TorchKernels(), weights="float8")
    with pytest.raises(ValueError, match="stored"):
        beholdd.Engine(folder, dtype="float32", max_tokens=64, device="cpu", kernels=TorchKernels(), weights="int4")
    with pytest.raises(ValueError, match="built model"):
        beholdd.Engine(model=object(), dtype="float32", max_tokens=64, device="cpu", kernels=TorchKernels(), weights="float8")
    out = io.StringIO()
    assert beholdd.cli.main(["generate", "--model", folder, "--weights", "int8", "--prompt-ids", "1"], out=out) != 0


def test_the_byte_plan_counts_what_is_kept(folder):
    """The layers' matrices in a byte a value with their scales; and the working memory of a step of many rows in 8 bits."""
    sizes = KernelSizes(verbose_build=False)
    kept = {}
    for weights in ("stored", "float8"):
        model, bound = open_model(folder, "bfloat16", "cpu", weights)
        bound.reader.close()
        kept[weights], transient = weights_as_kept(model, 2, sizes)
        assert transient > 0
    layers = sum(linear.in_features * linear.out_features for block in model.blocks
                 for linear in (block.mixer.qkv, block.mixer.out, block.feed_forward.gate_up, block.feed_forward.down))
    assert kept["stored"] - kept["float8"] > 0.3 * layers      # (small matrices are padded to whole blocks)
    assert sizes.gemm_float8_working_bytes(1, 4096, 4096, 2) == 8192
    assert sizes.gemm_float8_working_bytes(2048, 4096, 4096, 2) >= 2048 * 4096 * 3
    out = io.StringIO()
    assert beholdd.cli.main(["generate", "--model", folder, "--weights", "float8", "--plan-only", "--prompt-ids", "1,2"], out=out) == 0
    assert "weights:" in out.getvalue()


def _experts(**kw):
    part = RoutedExperts(32, 8, 2, 24, float("inf"), "m.", alpha=1.0, router_bias=False, scoring="sigmoid", shift=0.0, correction=True, groups=4,
                         keep_groups=2, factor=2.5, **kw)
    g = torch.Generator().manual_seed(5)
    tensors = {spec.name: torch.randn(spec.shape, generator=g) / 4 for spec in part.tensor_specs()}
    part.load(lambda name: tensors[name].clone())
    return part, tensors


def _context(kernels, rows):
    empty = torch.zeros(1, dtype=torch.int32)
    return StepContext(kernels=kernels, act_dtype=torch.float32, device=torch.device("cpu"), n_rows=rows, n_seqs=1, tokens=empty, positions=empty, row_seq=empty,
                       seq_start=empty, seq_slot=empty, seq_past=empty, host_seq_start=[0, rows], host_seq_slot=[0], host_seq_past=[0], is_decode=False,
                       max_position=rows)


@pytest.mark.parametrize("in_8_bits", [False, True])
def test_experts_behind_a_router_in_groups(in_8_bits):
    part, tensors = _experts()
    kernels = Float8TorchKernels()
    if in_8_bits:
        part.keep_in_float8()
    part.prepare(kernels)
    x = torch.randn((6, 32), generator=torch.Generator().manual_seed(1))
    out = torch.zeros((6, 32))
    ctx = _context(kernels, 6)
    part.forward(ctx, x, out)
    chosen, weights = plain.route(x @ tensors["m.router"].t(), tensors["m.correction"], 2, "sigmoid", 4, 2, "top2", True, 2.5)
    assert torch.equal(ctx.extras["routing"][0].long(), chosen)
    want = torch.zeros((6, 32), dtype=torch.float64)
    for r in range(6):
        for e, weight in zip(chosen[r].tolist(), weights[r].tolist()):
            g, u = (tensors[f"m.e{e}.{name}"].double() @ x[r].double() for name in ("gate", "up"))
            want[r] += weight * (tensors[f"m.e{e}.down"].double() @ (g * torch.sigmoid(g) * u))
    off = float((out.double() - want).norm() / want.norm())
    assert off < (0.15 if in_8_bits else 1e-5)


@pytest.mark.parametrize("kw", [dict(groups=3), dict(groups=4, keep_groups=5), dict(groups=8, keep_groups=1), dict(groups=4, scoring="softmax"),
                                dict(groups=4, group_score="sum"), dict(groups=4, router_bias=True)])
def test_groups_that_do_not_go(kw):
    with pytest.raises(ValueError):
        RoutedExperts(32, 8, 2, 24, 1.0, "m.", **{"router_bias": False, "scoring": "sigmoid", **kw})
