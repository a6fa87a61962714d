"""What the C entry points of the 8-bit products, the experts and the router in groups refuse before they launch anything, and the sizes
they say they need.  No GPU: every call here ends in an error or asks for a size."""

import ctypes

import pytest

from beholdd.kernels.library import Float8Rows, Float8Weight, KernelSizes


@pytest.fixture(scope="module")
def sizes():
    return KernelSizes(verbose_build=False)


AT = 4096      # an aligned address that nothing reads


@pytest.mark.parametrize("m,n,k,ldc,c_type,gate,at", [(0, 16, 128, 16, 0, 0, AT), (1, 0, 128, 16, 0, 0, AT), (1, 16, 0, 16, 0, 0, AT), (1, 16, 128, 15, 0, 0, AT),
                                                      (1, 16, 128, 16, 2, 0, AT), (1, 16, 128, 16, 0, 3, AT), (1, 16, 128, 16, 0, 0, AT + 8), (33, 16, 128, 16, 0, 0, AT)])
def test_products_refuse(sizes, m, n, k, ldc, c_type, gate, at):
    lib = sizes.lib
    assert lib.bh_gemm_float8_few(AT, 0, at, AT, AT, c_type, 0, m, n, k, ldc, gate, 1, None) != 0
    assert b"gemm_float8" in lib.bh_last_error()
    if m != 33:
        assert lib.bh_gemm_float8(AT, AT, at, AT, AT, c_type, 0, m, n, k, ldc, gate, 1, AT, None) != 0


def test_rows_refuse(sizes):
    lib = sizes.lib
    for rows, width, gate, dtype, at in ((0, 128, 0, 0, AT), (1, 0, 0, 0, AT), (1, 128, 7, 0, AT), (1, 128, 0, 5, AT), (1, 128, 0, 0, AT + 4)):
        assert lib.bh_float8_rows(AT, dtype, at, AT, rows, width, 0, gate, None) != 0


@pytest.mark.parametrize("n,stride,e,top,groups,keep", [(0, 16, 16, 1, 1, 1), (1, 15, 16, 1, 1, 1), (1, 2000, 1025, 1, 1, 1), (1, 16, 16, 0, 1, 1), (1, 16, 16, 17, 1, 1),
                                                        (1, 64, 64, 33, 1, 1), (1, 16, 16, 1, 3, 1), (1, 16, 16, 1, 4, 5), (1, 16, 16, 1, 4, 0), (1, 16, 16, 5, 4, 1),
                                                        (1, 130, 130, 1, 65, 1)])
def test_router_refuses(sizes, n, stride, e, top, groups, keep):
    assert sizes.lib.bh_route_in_groups(AT, stride, None, AT, AT, n, e, top, groups, keep, 0, 1, 1, 1.0, None) != 0
    assert b"route_in_groups" in sizes.lib.bh_last_error()


def test_experts_refuse(sizes):
    lib = sizes.lib
    assert lib.bh_experts_float8_rows(AT, 0, 1, AT, 0, 4, AT, AT, AT, 16, 128, 1, 1.0, 1.0, 0.0, None, 1, None) != 0
    assert lib.bh_experts_float8_rows(AT, 0, 1, AT, 1 << 20, 4, AT, AT, AT, 16, 128, 1, 1.0, 1.0, 0.0, None, 1, None) != 0
    assert lib.bh_experts_float8_rows(AT, 9, 1, AT, 4, 4, AT, AT, AT, 16, 128, 1, 1.0, 1.0, 0.0, None, 1, None) != 0
    assert lib.bh_experts_float8_tiles(AT, AT, 0, 1, AT, 4, AT, 4, 4, AT, AT, AT, AT, 16, 128, 1, 1.0, 1.0, 0.0, None, 1, None) != 0
    assert lib.bh_experts_float8_tiles(AT, AT, 4, 1, AT, 4, AT, 4, 4, AT + 1, AT, AT, AT, 16, 128, 1, 1.0, 1.0, 0.0, None, 1, None) != 0
    assert lib.bh_experts_float8_sum(AT, AT, AT, None, 0, AT, 0, 0, 4, 1, 128, 1, None) != 0
    assert lib.bh_experts_float8_sum(AT, AT, AT, None, 3, AT, 0, 4, 4, 1, 128, 1, None) != 0


def test_sizes():
    assert Float8Weight.data_bytes(2, 17, 129) == 2 * 32 * 256 and Float8Weight.scale_shape(2, 129, 129) == (2, 2, 2)
    assert Float8Rows.bytes_of(17, 513) == (32 * 640, 4 * 32 * 2)


def test_products_between_rows_in_8_bits_refuse(sizes):
    lib = sizes.lib
    assert lib.bh_gemm_float8_rows(AT, 0, None, AT, AT, AT, 0, 0, 40, 16, 128, 16, 0, 1, None) != 0
    assert lib.bh_gemm_float8_rows(AT, 7, AT, AT, AT, AT, 0, 0, 40, 16, 128, 16, 0, 1, None) != 0
    assert lib.bh_gemm_float8_rows(AT, 0, AT, AT + 8, AT, AT, 0, 0, 40, 16, 128, 16, 0, 1, None) != 0
    for m, n, k, gate, at in ((127, 256, 128, 1, AT), (400, 0, 128, 1, AT), (400, 256, 0, 1, AT), (400, 256, 128, 0, AT), (400, 256, 128, 9, AT), (400, 256, 128, 1, AT + 8)):
        assert lib.bh_gemm_float8_gated_to_8(AT, AT, at, AT, AT, AT, 0, m, n, k, gate, 1, None) != 0
        assert b"gemm_float8" in lib.bh_last_error()
    for rows, width, dtype, at in ((0, 128, 0, AT), (1, 0, 0, AT), (1, 8193, 0, AT), (1, 128, 5, AT), (1, 128, 0, AT + 4)):
        assert lib.bh_float8_norm(AT, AT, dtype, 1e-5, 0, at, AT, rows, width, None) != 0
        assert b"float8_norm" in lib.bh_last_error()


@pytest.mark.parametrize("n,k,gated", [(1024, 4096, False), (4096, 12288, False), (300, 5000, True)])
def test_the_plan_of_many_rows_counts_what_fewer_rows_take(sizes, n, k, gated):
    """K is cut into parts where the rows are few: a step of fewer rows than the plan's largest may need more for their sums."""
    planned = sizes.gemm_float8_working_bytes(1000, n, k, 2, gated)
    rows = sum(Float8Rows.bytes_of(1000, k))
    for m in range(17, 1001):
        for full in (0, 1):
            assert planned >= rows + sizes.lib.bh_gemm_float8_scratch(m, n, k, int(gated), full)
    assert max(sizes.lib.bh_gemm_float8_scratch(m, n, k, int(gated), 1) for m in range(17, 1000)) > sizes.lib.bh_gemm_float8_scratch(1000, n, k, int(gated), 1)
