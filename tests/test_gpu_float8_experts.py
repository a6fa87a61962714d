"""Experts whose matrices are kept in 8 bits: values that are not finite, and large ones, behind a limit."""

import math

import pytest
import torch

import plain_float8 as plain
from test_gpu_float8 import DEVICE, _close, _experts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k():
    from beholdd.kernels import HipKernels
    return HipKernels(DEVICE)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("more", [dict(limit=0.7, alpha=1.702, shift=1.0), dict(limit=7.0, weigh_input=True), dict()], ids=["clamped", "weighed", "plain"])
@pytest.mark.parametrize("n", [1, 2, 20, 200, 1000])
def test_a_value_that_is_not_finite_makes_its_row_nan_and_no_other(k, n, more, bad):
    """One row, few pairs, tiles of 64 and of 128 pairs: a limit on the gate and on up hides no broken value."""
    x, chosen, weights, packed, _ = _experts(k, n, 160, 64, 6, 2, torch.bfloat16, 3)
    out, whole = torch.empty((n, 160), device=DEVICE), torch.empty((n, 160), device=DEVICE)
    k.experts_float8(x.to(DEVICE), chosen.to(DEVICE), weights.to(DEVICE), *packed, whole, fresh=True, **more)
    x[n // 2, 7] = bad
    k.experts_float8(x.to(DEVICE), chosen.to(DEVICE), weights.to(DEVICE), *packed, out, fresh=True, **more)
    keep = [i for i in range(n) if i != n // 2]
    assert bool(torch.isnan(out[n // 2]).all()) and torch.equal(out[keep], whole[keep])


def test_the_clamp_is_as_it_was_for_numbers(k):
    """Sums beyond the limit on either side, of a row of large values."""
    x, chosen, weights, packed, held = _experts(k, 30, 200, 136, 5, 3, torch.float32, 9)
    x *= 50.0
    out = torch.full((30, 200), math.nan, device=DEVICE)
    more = dict(limit=0.7, alpha=1.702, shift=1.0)
    k.experts_float8(x.to(DEVICE), chosen.to(DEVICE), weights.to(DEVICE), *packed, out, fresh=True, **more)
    _close(out, *plain.experts(x, chosen, weights, *held, **more))
