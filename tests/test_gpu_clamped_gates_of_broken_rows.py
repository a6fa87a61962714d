"""A clamped gate hides no value that is not a number: every kernel that has one, with a broken row among others."""

import math

import pytest
import torch

from test_gpu_kernels import K, dev      # noqa: F401  (K: the fixture)

pytestmark = pytest.mark.gpu

ACT = dict(limit=0.7, alpha=1.702)


def _check(out, whole, bad):
    keep = [i for i in range(out.shape[0]) if i not in bad]
    assert bool(torch.isnan(out[bad]).all()) and torch.equal(out[keep], whole[keep]) and bool(torch.isfinite(whole).all())


def _twice(run, x, bad):
    """What `run` makes of the rows as they are and with a NaN in one."""
    whole = run(x)
    broken = x.clone()
    broken[bad, 5] = math.nan
    return run(broken), whole


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 40, 3000])
def test_the_activation(K, dtype, n):      # noqa: F811
    both = torch.randn(n, 128, generator=torch.Generator().manual_seed(1)).to(dtype)

    def run(rows):
        out = torch.empty(n, 64, dtype=dtype, device="cuda:0")
        K.clamped_glu(dev(rows), out, ACT["limit"], ACT["alpha"])
        return out

    whole = run(both)
    for column in (7, 64 + 7):      # the gate, and up
        broken = both.clone()
        broken[n // 2, column] = math.nan
        out = run(broken)
        assert bool(torch.isnan(out[n // 2, 7])) and int((out != whole).sum()) == 1


@pytest.mark.parametrize("n", [1, 20, 40, 300, 2100])
@pytest.mark.parametrize("ff", [64, 768])
def test_products(K, n, ff):      # noqa: F811
    g = torch.Generator().manual_seed(n)
    x, w = torch.randn(n, 1024, generator=g).to(torch.bfloat16), K.pack_weight(dev((torch.randn(2 * ff, 1024, generator=g) / 16).to(torch.bfloat16)))
    took = []

    def run(rows):
        out = torch.empty(n, ff, dtype=torch.bfloat16, device="cuda:0")
        took.append(K.gemm_clamped_glu(dev(rows), w, out, **ACT))
        return out

    out, whole = _twice(run, x, n // 2)
    if all(took):
        _check(out, whole, [n // 2])
    else:
        assert n > 32 and not any(took)      # (two launches, the second of them above)


@pytest.mark.parametrize("n", [1, 3, 40, 700])
@pytest.mark.parametrize("form", ["pairs", "rows", "tiles", "many"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_experts(K, n, form, dtype):      # noqa: F811
    """The inner values of a row's pairs."""
    if form in ("tiles", "many") and dtype != torch.bfloat16:
        return      # (kernels of bfloat16 alone)
    experts, top, width, ff = 4, 2, 128, 64
    g = torch.Generator().manual_seed(n)
    x, w = torch.randn(n, width, generator=g).to(dtype), dev((torch.randn(experts, 2 * ff, width, generator=g) / 8).to(dtype))
    chosen = dev(torch.rand(n, experts, generator=g).topk(top, dim=1).indices.to(torch.int32))
    lists, counts = torch.empty(experts, n, dtype=torch.int32, device="cuda:0"), torch.empty(experts, dtype=torch.int32, device="cuda:0")
    K.experts_group(chosen, lists, counts)
    packed = K.pack_weight(w.view(-1, width))

    def run(rows):
        inner = torch.empty(n * top, ff, dtype=dtype, device="cuda:0")
        if form == "pairs":
            K.experts_gate_up(dev(rows), chosen, w, inner, ACT["limit"], ACT["alpha"])
        else:
            product = {"rows": K.experts_rows, "tiles": K.experts_tiles, "many": K.experts_many}[form]
            product(dev(rows), top, lists, counts, w if form == "rows" else packed, inner, gated=True, **ACT)
        return inner

    out, whole = _twice(run, x, n // 2)
    _check(out, whole, [top * (n // 2) + j for j in range(top)])


def test_experts_of_a_prompt_in_stretches(K):      # noqa: F811
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(200, 128, generator=g).to(torch.bfloat16), dev((torch.randn(2, 128, 128, generator=g) / 8).to(torch.bfloat16))
    tiles = dev(torch.tensor([[0, 0, 100], [1, 100, 100]], dtype=torch.int32))

    def run(rows):
        out = torch.empty(200, 64, dtype=torch.bfloat16, device="cuda:0")
        K.experts_products(dev(rows), w, tiles, out, gated=True, **ACT)
        return out

    assert K.experts_products_take(torch.bfloat16, 128, 128)
    _check(*_twice(run, x, 130), [130])
