"""The byte plan of engines with 8-bit weights against what is allocated while they load and run."""

import pytest
import torch

import beholdd
from test_float8_plan import folders, sizes      # noqa: F401 (fixtures)
from test_float8_plan import _plan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["dense", "experts"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_the_plan_bounds_what_is_allocated(folders, which, dtype):      # noqa: F811
    """A limit that the stored weights exceed: in 8 bits the engine loads and runs within it, and holds what its plan says beside the steps."""
    options = dict(dtype=dtype, max_tokens=2048, max_slots=4, max_rows_per_step=500, device="cuda:0")
    stored = beholdd.Engine(folders[which], **options).plan.total_bytes
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(beholdd.MemoryBudgetError):
        beholdd.Engine(folders[which], memory_limit_bytes=stored - 1, **options)
    assert torch.cuda.max_memory_allocated() == before
    engine = beholdd.Engine(folders[which], weights="float8", memory_limit_bytes=stored - 1, **options)
    loading = torch.cuda.max_memory_allocated() - before
    assert loading <= sum(engine.plan.bytes_of(label) for label, _ in engine.plan.items if label.startswith(("weights", "largest transient", "tables", "cache", "sampler")))
    slots = [engine.alloc_slot() for _ in range(2)]
    engine.step([beholdd.StepEntry(slots[0], [3] * 490, [489]), beholdd.StepEntry(slots[1], [4] * 7, [6])])
    for _ in range(4):
        engine.step([beholdd.StepEntry(slot, [7], [0]) for slot in slots])
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before <= engine.plan.total_bytes < stored


def test_a_float32_file_in_a_bfloat16_engine(tmp_path):
    """Its layers stand in four bytes a value until they are in 8 bits."""
    from test_float8_plan import WIDE
    beholdd.write_random_model(str(tmp_path), dict(WIDE, num_hidden_layers=2), seed=1, dtype="float32", std=0.05)
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    engine = beholdd.Engine(str(tmp_path), dtype="bfloat16", max_tokens=256, max_slots=2, device="cuda:0", weights="float8")
    engine.step([beholdd.StepEntry(engine.alloc_slot(), [3] * 200, [199])])
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before <= engine.plan.total_bytes
