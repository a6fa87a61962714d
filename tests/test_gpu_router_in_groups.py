"""A model whose configuration names the feed-forward of experts in groups, on the GPU, against the same engine over 64-bit kernels on the CPU."""

import pytest
import torch

import beholdd
import models_of_groups as models
from float8_emulation import Float8TorchKernels
from test_gpu_float8_models import EACH

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weights", ["stored", "float8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_model_with_experts_in_groups(tmp_path, weights, dtype):
    """A prompt, captured single tokens behind it and a batch.  Stored weights: float32 sums of some hundred terms in a dozen products, 1e-4 of the
    logits; bfloat16 roundings of 2^-9 in some ten places a layer, 2 % of three layers' logits by norm.  In 8 bits what falls on the other side of a
    border, as for every architecture.  The median position, for a choice next to a border may go another way."""
    folder = models.folder(str(tmp_path), dtype)      # (stored experts are multiplied in the file's type)
    tokens, rows = [int(t) for t in torch.randint(0, 301, (60,), generator=torch.Generator().manual_seed(2))], []
    for device, kernels in (("cuda:0", None), ("cpu", Float8TorchKernels())):
        engine = beholdd.Engine(folder, dtype=dtype, max_tokens=512, device=device, kernels=kernels, weights=weights)
        slot, got = engine.alloc_slot(), []
        for first, last in ((0, 40), (40, 50), *((t, t + 1) for t in range(50, 60))):
            got.append(engine.step([beholdd.StepEntry(slot, tokens[first:last], list(range(last - first)))]).float().cpu())
        rows.append(torch.cat(got))
    models.unregister()
    off = (rows[0] - rows[1]).norm(dim=1) / rows[1].norm(dim=1)
    bound = {"float32": 1e-4, "bfloat16": 0.02}[dtype] if weights == "stored" else 1.5 * EACH[dtype] * (4.0 * models.CONFIG["num_hidden_layers"]) ** 0.5
    assert bool(torch.isfinite(rows[0]).all()) and float(off.median()) < bound
