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
