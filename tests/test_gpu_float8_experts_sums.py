"""How the products of experts whose matrices are kept in 8 bits add up: gate and up in full, down as it is said."""

import math

import pytest
import torch

import plain_float8 as plain
from test_gpu_float8 import DEVICE, EXPERTS, _close, _experts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k():
    from beholdd.kernels import HipKernels
    return HipKernels(DEVICE)


@pytest.mark.parametrize("n,top,experts", [(1, 2, 4), (3, 2, 4), (40, 2, 4), (300, 2, 3), (300, 4, 20)])
@pytest.mark.parametrize("full", [None, False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gate_and_up_sums_are_full(k, n, top, experts, full, dtype):
    """Two products of 448^2 that cancel and six of 1 beside them, eight neighbouring k in all: 6 in full, and nothing of them where what lies 2^14
    below the largest of eight is dropped.  silu(6) * 6 = 35.9 is 36 in 8 bits, whatever the exponential's rounding, and stands alone in its row of `down`."""
    x = torch.zeros((n, 128))
    x[:, :8] = torch.tensor([448.0, 448.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0])
    row = torch.zeros(128)
    row[:8] = torch.tensor([448.0, -448.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0])
    ff, width = 128, 128
    up = row.repeat(2 * experts * ff, 1).to(torch.float8_e4m3fn)
    down = torch.eye(width).repeat(experts, 1).to(torch.float8_e4m3fn)
    w_up = k.pack_float8(up.to(DEVICE), torch.ones((2 * experts, 1, 1), device=DEVICE))
    w_down = k.pack_float8(down.to(DEVICE), torch.ones((experts, 1, 1), device=DEVICE))
    chosen = torch.randint(0, experts, (n, top), generator=torch.Generator().manual_seed(n), dtype=torch.int32)
    out = torch.full((n, width), math.nan, device=DEVICE)
    k.experts_float8(x.to(dtype).to(DEVICE), chosen.to(DEVICE), torch.full((n, top), 0.5, device=DEVICE), w_up, w_down, out, fresh=True, full_sums=full)
    assert torch.equal(out.cpu(), torch.full((n, width), 0.5 * top * 36.0))


@pytest.mark.parametrize("n,width,ff,e,top", EXPERTS)
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("full", [False, True])
def test_how_the_down_product_adds_up(k, n, width, ff, e, top, out_dtype, full):
    x, chosen, weights, packed, held = _experts(k, n, width, ff, e, top, torch.bfloat16, n + e)
    out = torch.full((n, width), math.nan, dtype=out_dtype, device=DEVICE)
    k.experts_float8(x.to(DEVICE), chosen.to(DEVICE), weights.to(DEVICE), *packed, out, fresh=True, full_sums=full)
    _close(out, *plain.experts(x, chosen, weights, *held, full=full))
