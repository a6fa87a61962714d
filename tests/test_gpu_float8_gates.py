"""Gated products with 8-bit weights and float32 outputs are within float32's errors of the gate's activation, wherever the gate lies."""

import math

import pytest
import torch

from test_gpu_float8 import DEVICE

pytestmark = pytest.mark.gpu

# Every e4m3 value with at least an eighth in magnitude, up to 88 (beyond which exp(-y) is none of float32's numbers): 4 significant bits.
VALUES = sorted({s * m * 2.0 ** e for s in (-1.0, 1.0) for m in (1.0, 1.125, 1.25, 1.375, 1.5, 1.625, 1.75, 1.875) for e in range(-3, 7) if m * 2.0 ** e <= 88.0})


@pytest.fixture(scope="module")
def k():
    from beholdd.kernels import HipKernels
    return HipKernels(DEVICE)


@pytest.mark.parametrize("m,width,repeats", [(1, 256, 1), (16, 256, 1), (40, 256, 2), (70, 256, 1), (200, 256, 1), (200, 4096, 3), (2500, 512, 8)])
@pytest.mark.parametrize("full", [None, False])
def test_gate_of_a_float32_output(k, m, width, repeats, full):
    """Gate and up sums are exact: every output has a single product of e4m3 numbers in each.  What is left are the exponential (a unit in the last
    place at most), one addition, one division and the product with 1: 2^-23 + 2^-24 + 2^-24 = 2^-22 of the value."""
    count = len(VALUES)
    assert count < 255
    x = torch.zeros((m, width))
    x[:, 0] = 1.0
    x[:, 1:1 + count] = torch.tensor(VALUES)
    x = torch.where(torch.arange(m)[:, None] % 2 == 0, x, x * torch.where(torch.arange(width) == 0, 1.0, -1.0))
    n = repeats * count
    w = torch.zeros((2 * n, width))
    w[torch.arange(n), 1 + torch.arange(n) % count] = 1.0
    w[n:, 0] = 1.0
    scales = torch.ones((2, -(-n // 128), -(-width // 128)))
    weight = k.pack_float8(w.to(torch.float8_e4m3fn).to(DEVICE), scales.to(DEVICE))
    out = torch.full((m, n), math.nan, device=DEVICE)
    k.gemm_swiglu(x.to(DEVICE), weight, out, full_sums=full)
    y = x[:, 1:1 + count].double().repeat(1, repeats)
    want = y / (1.0 + torch.exp(-y))
    off = (out.double().cpu() - want).abs() / want.abs()
    assert off.max().item() <= 2.0 ** -22, f"{off.max().item():.3e} at {y.flatten()[off.flatten().argmax()].item()}"
