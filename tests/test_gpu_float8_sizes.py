"""Products with 8-bit weights on every kernel that a call can reach, with outputs of both types, written and added, against their definition in 64
bits.  Which sizes reach which kernel is asserted without a GPU (test_float8_dispatch.py)."""

import math

import pytest
import torch

import plain_float8 as plain
from float8_sizes import SIZES
from test_gpu_float8 import DEVICE, _close, _rows, _weight

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k():
    from beholdd.kernels import HipKernels
    return HipKernels(DEVICE)


@pytest.mark.parametrize("key", list(SIZES), ids=str)
def test_product(k, key):
    (rows_type, *_), gated, full = key
    m, n, width = SIZES[key]
    x, (w, held) = _rows(m, width, torch.float32 if rows_type == "float32" else torch.bfloat16, m + width), _weight(k, 2 if gated else 1, n, width, 2)
    a = x.to(DEVICE)
    if rows_type == "float8" and m <= 16:      # (more rows are brought into 8 bits in the call)
        a = k.to_float8(a)
    pick = sorted({0, 1 % m, 15 % m, 16 % m, 31 % m, 32 % m, 63 % m, 64 % m, 127 % m, 128 % m, m // 2, (m - 2) % m, m - 1})
    x8, whole = plain.rows(x[pick]), plain.matrix(*held)
    if gated:
        want, bound = plain.gated(*plain.product(x8, whole[:n], full), *plain.product(x8, whole[n:], full))
    else:
        want, bound = plain.product(x8, whole, full)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((m, n), math.nan, dtype=dtype, device=DEVICE)
        (k.gemm_swiglu if gated else k.gemm)(a, w, out, full_sums=full)
        _close(out[pick], want, bound, f"{dtype}")
        assert bool(torch.isfinite(out).all())
        if not gated:
            before = torch.randn((m, n), generator=torch.Generator().manual_seed(3)).to(dtype)
            out.copy_(before)
            k.gemm(a, w, out, accumulate=True, full_sums=full)
            old = before[pick].double()
            _close(out[pick], want + old, bound + 2.0 ** -24 * (want.abs() + old.abs()), f"{dtype}, added")
            assert bool(torch.isfinite(out).all())
