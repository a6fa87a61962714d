"""A model whose configuration names the feed-forward of experts in groups, on the GPU, against the same engine over 64-bit kernels on the CPU."""

import pytest
import torch

import beholdd
import models_of_groups as models
from float8_emulation import Float8TorchKernels
from test_gpu_float8_models import EACH

pytestmark = pytest.mark.gpu


class Following(Float8TorchKernels):
    """Takes the choices that another engine made, in turn, and weighs them by its own scores: a choice next to a border goes either way, and a
    position that goes another way changes every later one, which looks back at it."""

    def __init__(self, choices):
        super().__init__()
        self.choices, self.apart = iter(choices), 0

    def route_in_groups(self, logits, correction, chosen, weights, scoring="sigmoid", groups=1, keep=None, group_score="top2", renorm=True, factor=1.0, experts=None):
        super().route_in_groups(logits, correction, chosen, weights, scoring, groups, keep, group_score, renorm, factor, experts)
        theirs = next(self.choices)
        self.apart += int((theirs != chosen).any(dim=1).sum())
        chosen.copy_(theirs)
        scores = torch.gather(torch.sigmoid(logits[:, :experts].double()), 1, chosen.long())
        weights.copy_((scores / scores.sum(dim=1, keepdim=True) * factor).float())


@pytest.mark.parametrize("weights", ["stored", "float8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_model_with_experts_in_groups(tmp_path, weights, dtype):
    """A prompt, a portion and single tokens.  Stored weights: float32 sums of some hundred terms in a dozen products, 1e-4 of the
    logits; bfloat16 roundings of 2^-9 in some ten places a layer, 2 % of three layers' logits by norm.  In 8 bits what falls on the other side of a
    border, as for every architecture.  Neighbours among the largest of 16 scores lie a quarter of their spread apart, and five such distances decide a
    row's choices and their order: float32's 1e-4 turn one row in some hundred, the other forms' errors one in a few, which says nothing."""
    folder = models.folder(str(tmp_path), dtype)      # (stored experts are multiplied in the file's type)
    tokens, rows, choices = [int(t) for t in torch.randint(0, 301, (60,), generator=torch.Generator().manual_seed(2))], [], []
    for device in ("cuda:0", "cpu"):
        kernels = Following(choices) if device == "cpu" else None
        engine = beholdd.Engine(folder, dtype=dtype, max_tokens=512, device=device, kernels=kernels, weights=weights, use_graphs=False)
        if kernels is None:
            real = engine.kernels.route_in_groups

            def route(logits, correction, chosen, *args, **kw):
                real(logits, correction, chosen, *args, **kw)
                choices.append(chosen.cpu())

            engine.kernels.route_in_groups = route
        slot, got = engine.alloc_slot(), []
        for first, last in ((0, 40), (40, 50), *((t, t + 1) for t in range(50, 60))):
            got.append(engine.step([beholdd.StepEntry(slot, tokens[first:last], list(range(last - first)))]).float().cpu())
        rows.append(torch.cat(got))
    models.unregister()
    assert len(choices) == 3 * 12
    if weights == "stored" and dtype == "float32":
        assert kernels.apart <= 3 * 60 // 10
    off = (rows[0] - rows[1]).norm(dim=1) / rows[1].norm(dim=1)
    bound = {"float32": 1e-4, "bfloat16": 0.02}[dtype] if weights == "stored" else 1.5 * EACH[dtype] * (4.0 * models.CONFIG["num_hidden_layers"]) ** 0.5
    assert bool(torch.isfinite(rows[0]).all()) and float(off.median()) < bound


@pytest.mark.parametrize("weights", ["stored", "float8"])
def test_captured_steps_are_the_eager_ones(tmp_path, weights):
    """Single tokens of three sequences replayed, with eager steps between, bit by bit as an engine without captures makes them."""
    folder, got = models.folder(str(tmp_path), "bfloat16"), []
    for graphs in (True, False):
        engine = beholdd.Engine(folder, dtype="bfloat16", max_tokens=1024, max_slots=4, device="cuda:0", weights=weights, use_graphs=graphs)
        slots, rows = [engine.alloc_slot() for _ in range(3)], []
        engine.step([beholdd.StepEntry(slot, list(range(5 + slot)), [0]) for slot in slots])
        for t in range(5):
            rows.append(engine.step([beholdd.StepEntry(slot, [7 * t + slot], [0]) for slot in slots]).clone())
            other = engine.alloc_slot()
            engine.step([beholdd.StepEntry(other, [1, 2, 3, t], [3])])
            engine.free_slot(other)
            torch.cuda.synchronize()
        got.append(torch.cat(rows))
    models.unregister()
    assert torch.equal(got[0], got[1])
