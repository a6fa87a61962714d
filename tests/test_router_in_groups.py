"""A model whose configuration names the feed-forward of experts in groups: built, loaded and run through the engine.  On the CPU."""

import pytest
import torch

import beholdd
import models_of_groups as models
import plain_float8 as plain
from float8_emulation import Float8TorchKernels


@pytest.fixture()
def folder(tmp_path):
    yield models.folder(str(tmp_path))
    models.unregister()


@pytest.mark.parametrize("weights", ["stored", "float8"])
def test_a_model_with_experts_in_groups(folder, weights):
    """Portions and single tokens give a whole prompt's logits, the choices are those of the definition, and the shared expert counts."""
    kernels = Float8TorchKernels()
    engine = beholdd.Engine(folder, dtype="float32", max_tokens=256, device="cpu", kernels=kernels, weights=weights)
    sizes, part = models.SIZES, engine.model.own_blocks()[-1].feed_forward
    assert (part.n_experts, part.top, part.ff, part.groups, part.keep_groups, part.factor) == (
        sizes.experts, sizes.top, sizes.expert_ff, sizes.groups, sizes.keep_groups, sizes.factor)
    assert part.shared.intermediate == sizes.shared_ff and part.has_correction and part.renorm and part.scoring == "sigmoid" and not part.has_router_bias
    tokens, extras, seen = [3, 1, 4, 1, 5, 9, 2, 6, 5, 3], {}, []
    real = kernels.route_in_groups
    kernels.route_in_groups = lambda logits, *args, **kw: (seen.append((logits[:, :kw["experts"]].clone(), args[0].clone(), kw)), real(logits, *args, **kw))
    whole = engine.step([beholdd.StepEntry(engine.alloc_slot(), tokens, list(range(10)))], extras)
    assert len(seen) == 3      # a layer each
    logits, correction, kw = seen[-1]
    chosen, weights_of = plain.route(logits, correction, sizes.top, "sigmoid", sizes.groups, sizes.keep_groups, "top2", True, sizes.factor)
    assert torch.equal(extras["routing"][0].long(), chosen) and torch.allclose(extras["routing"][1].double(), weights_of, rtol=1e-6)
    assert kw["groups"] == sizes.groups and kw["keep"] == sizes.keep_groups and kw["factor"] == sizes.factor
    slot = engine.alloc_slot()
    rows = [engine.step([beholdd.StepEntry(slot, tokens[:6], list(range(6)))])] + [engine.step([beholdd.StepEntry(slot, [t], [0])]) for t in tokens[6:]]
    assert torch.allclose(torch.cat(rows), whole, rtol=0.0, atol=float(whole.abs().max()) * 2e-5)
    part.shared.down.weight = part.shared.down.weight * 0.0 if weights == "stored" else part.shared.down.weight
    if weights == "stored":
        assert not torch.allclose(engine.step([beholdd.StepEntry(engine.alloc_slot(), tokens, list(range(10)))]), whole, atol=1e-3)
    assert (kernels.products > 0) == (weights == "float8")
