"""Which kernel a product with an 8-bit weight runs on: that the sizes the GPU tests compare reach every one of them, and that no call reaches another.
No GPU: the library answers from sizes."""

import math
import random

import pytest

from beholdd.kernels.library import KernelSizes
from float8_sizes import SIZES, form


@pytest.fixture(scope="module")
def lib():
    return KernelSizes(verbose_build=False).lib


@pytest.mark.parametrize("key", list(SIZES), ids=str)
def test_each_size_runs_on_the_kernel_it_stands_for(lib, key):
    (rows_type, *_), gated, full = key
    assert form(lib, rows_type, *SIZES[key], gated, full) == key


@pytest.mark.parametrize("gated,full", [(False, False), (False, True), (True, False), (True, True)])
def test_no_call_runs_on_another(lib, gated, full):
    """Thousands of sizes, spread over their logarithms."""
    rng = random.Random(7)
    between = lambda low, high: round(math.exp(rng.uniform(math.log(low), math.log(high))))
    for _ in range(20000):
        m, n, k = between(1, 9000), between(16, 14000), between(1, 13000)
        if rng.random() < 0.5:
            k = max(128, k // 128 * 128)
        for rows_type in ("float8", "float32", "bfloat16") if m <= 16 else ("float8",):
            assert form(lib, rows_type, m, n, k, gated, full) in SIZES, (rows_type, m, n, k)


def test_gated_products_of_a_prompt_leave_their_rows_in_8_bits(lib):
    """The sizes whose comparison with `gemm_swiglu` on the GPU would say nothing if the rule took none of them."""
    for m, n, k in ((128, 12288, 4096), (2048, 12288, 4096), (8192, 12288, 4096), (400, 4100, 130), (130, 700, 300), (700, 12288, 512), (1000, 4100, 1000)):
        assert lib.bh_gemm_float8_gives_8(m, n, k, 0) == 1
    for m, n, k in ((512, 12288, 4096), (2048, 12288, 4096), (400, 4100, 130), (5000, 300, 130)):
        assert lib.bh_gemm_float8_gives_8(m, n, k, 1) == 1
    assert lib.bh_gemm_float8_gives_8(127, 12288, 4096, 0) == 0


def test_refusals(lib):
    import ctypes
    kernel = (ctypes.c_int * 4)()
    for m, n, k, to in ((0, 16, 128, kernel), (1, 0, 128, kernel), (1, 16, 0, kernel), (1, 16, 128, None)):
        assert lib.bh_gemm_float8_kernel(-1, m, n, k, 0, 0, to) != 0


def test_gate_and_up_sums_of_experts_are_full(lib):
    """The C entries refuse to make them otherwise, before anything is launched."""
    at = 4096
    assert lib.bh_experts_float8_rows(at, 0, 1, at, 4, 4, at, at, at, 16, 128, 1, 1.0, 1.0, 0.0, None, 0, None) != 0
    assert b"in full" in lib.bh_last_error()
    assert lib.bh_experts_float8_tiles(at, at, 4, 1, at, 4, at, 4, 4, at, at, at, at, 16, 128, 1, 1.0, 1.0, 0.0, None, 0, None) != 0
    assert b"in full" in lib.bh_last_error()
