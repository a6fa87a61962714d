"""Norms and gated products that write rows in 8 bits do so only where everything that reads them takes such rows: every configuration of every
architecture over kernels that have these forms, whose rows in 8 bits nothing but a product with an 8-bit weight can read.  On the CPU."""

import importlib

import numpy as np
import pytest
import torch

import beholdd
import conftest
import plain_float8 as plain
from float8_emulation import Float8Matrix, Float8TorchKernels


class RowsIn8:
    """What the library's `Float8Rows` are to the parts: a matrix's shape, and nothing that another operation could read."""

    def __init__(self, values):
        self.values, self.shape, self.dtype, self.device = values, values.shape, torch.float8_e4m3fn, values.device

    def dim(self):
        return 2


class KernelsThatWriteRowsIn8(Float8TorchKernels):
    """A value that was rounded to 8 bits once stays what it is, so results are those of `Float8TorchKernels`."""
    FEW_ROWS = 16

    def __init__(self):
        super().__init__()
        self.norms = self.gated = 0

    def rmsnorm_float8(self, x, weight, eps, dtype=torch.float32):
        if x.shape[0] <= self.FEW_ROWS:
            return None
        self.norms += 1
        out = torch.empty(x.shape, dtype=dtype)
        self.rmsnorm(x, weight, eps, out)
        return RowsIn8(plain.rows(out))

    def gemm_swiglu_float8(self, a, w, gate="silu", dtype=torch.float32):
        assert isinstance(w, Float8Matrix) and w.matrices == 2
        if a.shape[0] <= self.FEW_ROWS:
            return None
        self.gated += 1
        out = torch.empty((a.shape[0], w.shape[0] // 2), dtype=dtype)
        self.gemm_swiglu(a, w, out, gate)
        return RowsIn8(plain.rows(out))

    @staticmethod
    def _taken(a, w):
        if isinstance(a, RowsIn8):
            assert isinstance(w, Float8Matrix), "rows in 8 bits went into a product with a stored weight"
            return a.values
        return a

    def gemm(self, a, w, out, accumulate=False, then_norm=None, full_sums=None):
        return super().gemm(self._taken(a, w), w, out, accumulate, then_norm, full_sums)

    def gemm_swiglu(self, a, w, out, gate="silu"):
        return super().gemm_swiglu(self._taken(a, w), w, out, gate)


def _folder(name, which, path):
    if name == "qwen3":
        beholdd.write_random_model(path, conftest.CONFIGS[which], seed=2, dtype="float32", std=0.1)
    else:
        models = importlib.import_module(f"{name}_models")
        models.write_model(path, models.CONFIGS[which], models.random_weights(models.CONFIGS[which], seed=5))
    return path


MODELS = [("qwen3", which) for which in sorted(conftest.CONFIGS)]
for _name in ("dupidra", "gokazen", "lurepel", "pudorax", "vepelix", "vitudra"):
    MODELS += [(_name, which) for which in importlib.import_module(f"{_name}_models").CONFIGS]


@pytest.mark.parametrize("name,which", MODELS)
def test_rows_in_8_bits_go_to_products_alone(name, which, tmp_path):
    """A prompt of more rows than products take as they are, and single tokens behind it, as without these forms."""
    folder, got = _folder(name, which, str(tmp_path)), []
    for kernels in (Float8TorchKernels(), KernelsThatWriteRowsIn8()):
        engine = beholdd.Engine(folder, dtype="float32", max_tokens=256, device="cpu", kernels=kernels, weights="float8")
        tokens = [int(t) for t in np.random.default_rng(6).integers(0, engine.model.vocab, size=26)]
        slot = engine.alloc_slot()
        rows = [engine.step([beholdd.StepEntry(slot, tokens[:24], list(range(24)))])]
        rows += [engine.step([beholdd.StepEntry(slot, [token], [0])]) for token in tokens[24:]]
        got.append(torch.cat(rows))
    assert bool(torch.isfinite(got[0]).all())
    assert torch.equal(got[1], got[0])


def test_the_forms_are_used(tmp_path):
    """So that the comparison above says something: a layer's two norms and its gated product, in the prompt alone."""
    engine = beholdd.Engine(_folder("qwen3", "A", str(tmp_path)), dtype="float32", max_tokens=256, device="cpu", kernels=KernelsThatWriteRowsIn8(), weights="float8")
    slot, layers = engine.alloc_slot(), len(engine.model.blocks)
    engine.step([beholdd.StepEntry(slot, [3] * 24, [23])])
    assert (engine.kernels.norms, engine.kernels.gated) == (2 * layers, layers)
    engine.step([beholdd.StepEntry(slot, [3], [0])])
    assert (engine.kernels.norms, engine.kernels.gated) == (2 * layers, layers)
