"""What engines with 8-bit weights plan to allocate, without a GPU."""

import math
import random

import pytest

from beholdd.engine.memory import step_size
from beholdd.kernels.library import Float8Rows, KernelSizes
from beholdd.parts.experts import RoutedExperts


@pytest.fixture(scope="module")
def sizes():
    return KernelSizes(verbose_build=False)


def _unit(n_bytes):
    return -(-n_bytes // 512) * 512


def _experts_allocate(lib, n, top, experts, width, ff):
    """The tensors of one call of `experts_float8`, as it makes them."""
    pairs = n * top
    if lib.bh_experts_float8_one(pairs, top):
        return _unit(4 * pairs * ff)
    results = _unit(4 * pairs * width)
    if lib.bh_experts_float8_few(pairs, experts):
        return results + _unit(4 * pairs * ff)
    return (results + _unit(4 * experts * pairs) + _unit(4 * experts) + sum(map(_unit, Float8Rows.bytes_of(n, width))) + sum(map(_unit, Float8Rows.bytes_of(pairs, ff))))


def _experts_cases():
    rng = random.Random(3)
    between = lambda low, high: round(math.exp(rng.uniform(math.log(low), math.log(high))))
    yield 4096, 8, 32, 64, 8
    for _ in range(200):
        yield between(1, 5000), rng.randint(1, 12), between(1, 200), between(1, 3000), between(1, 2000)


def test_experts_plan_what_they_allocate(sizes):
    """For the planned number of rows and for fewer, narrow experts among them, whose rows in 8 bits have whole stretches."""
    for n, top, experts, width, ff in _experts_cases():
        planned = sizes.experts_float8_working_bytes(n, top, experts, width, ff)
        for rows in sorted({1, min(2, n), n // 3 + 1, max(n - 1, 1), n, *(min(max(count // top, 1), n) for count in (32, 128, 1000, 1024, 1030, 8 * experts, 8 * experts + top))}):
            assert _experts_allocate(sizes.lib, rows, top, experts, width, ff) <= planned, (rows, n, top, experts, width, ff)


@pytest.mark.parametrize("rows", [1, 300, 4096])
def test_the_part_plans_its_experts(sizes, rows):
    part = RoutedExperts(64, 32, 8, 8, float("inf"), "m.", router_bias=False)
    part.keep_in_float8()
    step = step_size(type("Model", (), {}), rows, 1, 2, 8192, sizes)
    # the router's logits (kept 128 wide where the rows are many), the choices and their weights, the input in another form
    beside = _unit(4 * rows * (128 if rows > 32 else 32)) + 2 * _unit(4 * rows * 8) + _unit(2 * rows * 64)
    assert part.working_bytes(step) >= _experts_allocate(sizes.lib, rows, 8, 32, 64, 8) + beside
