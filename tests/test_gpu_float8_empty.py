"""Rows without a value, and no rows, are refused as other calls are that the kernels do not take; calls without weights."""

import math

import pytest
import torch

import plain_float8 as plain
from test_gpu_float8 import DEVICE, _close, _experts, _weight

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k():
    from beholdd.kernels import HipKernels
    return HipKernels(DEVICE)


@pytest.mark.parametrize("shape", [(4, 0), (0, 4), (0, 0), (20, 0)])
def test_rows_without_a_value(k, shape):
    from beholdd.kernels.library import KernelError
    x = torch.empty(shape, device=DEVICE)
    for call in (lambda: k.to_float8(x), lambda: k.to_float8(x, in_rows=True), lambda: k.to_float8(x, gate="silu")):
        with pytest.raises(KernelError):
            call()
    if shape[0] > 16:
        with pytest.raises(KernelError):
            k.rmsnorm_float8(x, None, 1e-5)


def test_products_without_a_row(k):
    from beholdd.kernels.library import KernelError
    w = _weight(k, 2, 16, 128, 1)[0]
    with pytest.raises(KernelError):
        k.gemm(torch.empty((0, 128), device=DEVICE), w, torch.empty((0, 32), device=DEVICE))
    with pytest.raises(KernelError):
        k.gemm_swiglu(torch.empty((0, 128), device=DEVICE), w, torch.empty((0, 16), device=DEVICE))


@pytest.mark.parametrize("n", [1, 20, 200])
def test_experts_without_weights(k, n):
    """Every pair counts once."""
    x, chosen, _, packed, held = _experts(k, n, 200, 136, 5, 3, torch.bfloat16, 9)
    out = torch.full((n, 200), math.nan, device=DEVICE)
    k.experts_float8(x.to(DEVICE), chosen.to(DEVICE), None, *packed, out, fresh=True)
    _close(out, *plain.experts(x, chosen, None, *held))
