"""Every configuration of every architecture with its layers' matrices in 8 bits, on the GPU, against the same engine over 64-bit kernels on the CPU."""

import numpy as np
import pytest
import torch

import beholdd
from float8_emulation import Float8TorchKernels
from test_float8_readers import MODELS, _folder

pytestmark = pytest.mark.gpu

# A value that falls on the other side of a border between two e4m3 numbers is 2^-3 of itself off.  In float32 at most one in a thousand does, which is
# 0.4 % of a product's input by norm; in bfloat16, 2^-9 off in each of some ten roundings a layer, one in sixteen, 3.2 %.  A layer has about four
# products one behind the other, and their errors add up as squares do.  Half as much again for what is not a product.
EACH = {"float32": 0.004, "bfloat16": 0.032}


@pytest.mark.parametrize("name,which", MODELS)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_model(name, which, dtype, tmp_path):
    """A prompt of more rows than products take as they are, one of fewer, and single tokens: the median position (a choice of experts next to a border
    may go another way, and a position with it)."""
    folder, rows = _folder(name, which, str(tmp_path)), []
    for device, kernels in (("cuda:0", None), ("cpu", Float8TorchKernels())):
        engine = beholdd.Engine(folder, dtype=dtype, max_tokens=1024, device=device, kernels=kernels, weights="float8")
        tokens = [int(t) for t in np.random.default_rng(6).integers(0, engine.model.vocab, size=60)]
        slot, got = engine.alloc_slot(), []
        for first, last in ((0, 40), (40, 52), *((t, t + 1) for t in range(52, 60))):
            got.append(engine.step([beholdd.StepEntry(slot, tokens[first:last], list(range(last - first)))]).float().cpu())
        rows.append(torch.cat(got))
    got, want = rows
    assert bool(torch.isfinite(got).all())
    off = (got - want).norm(dim=1) / want.norm(dim=1)
    assert float(off.median()) < 1.5 * EACH[dtype] * (4.0 * len(engine.model.schedule)) ** 0.5
