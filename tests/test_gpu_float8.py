"""Products with weights in 8 bits, experts in 8 bits and the router in groups, against their definitions in 64 bits."""

import math

import pytest
import torch

import plain_float8 as plain

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"


@pytest.fixture(scope="module")
def k():
    from beholdd.kernels import HipKernels
    return HipKernels(DEVICE)


def _rows(n, width, dtype, seed):
    """Rows of several sizes with a few large channels, and one of zeros where there are three or more."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, width), generator=g) * torch.exp(torch.randn((n, 1), generator=g))
    x *= 1.0 + 15.0 * (torch.rand(width, generator=g) < 0.02)
    if n > 2:
        x[n // 2] = 0.0
    return x.to(dtype)


def _weight(k, matrices, n, width, seed):
    """(a packed weight, its values and scales) that stand for the same."""
    g = torch.Generator().manual_seed(seed)
    w = torch.randn((matrices * n, width), generator=g) / math.sqrt(width) * (1.0 + torch.rand((matrices * n, 1), generator=g))
    return k.pack_float8(w.to(DEVICE), matrices=matrices), plain.quantised_matrix(w, matrices)


def _close(got, want, bound, what=""):
    """Within the bound of the sums and half a step of the output's type."""
    allowed = bound + plain.HALF_STEP[got.dtype] * (want.abs() + bound)
    off = (got.double().cpu() - want).abs()
    worst = (off - allowed).max().item()
    assert worst <= 0.0, f"{what}: off by {off.max().item():.3e}, {worst:.3e} more than allowed"


# ---- rows and weights in 8 bits ------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,width", [(1, 1), (3, 127), (16, 128), (17, 129), (5, 513), (40, 1000), (129, 4096)])
@pytest.mark.parametrize("in_rows", [False, True])
def test_rows_in_8_bits(k, dtype, n, width, in_rows):
    x = _rows(n, width, dtype, n + width)
    assert torch.equal(k.from_float8(k.to_float8(x.to(DEVICE), in_rows=in_rows)).double().cpu(), plain.rows(x))


def test_rows_in_8_bits_at_the_borders(k):
    """Ties go to even, 448 itself to 448 of its scale, what is larger to the next scale; magnitudes from the smallest to the largest."""
    steps = torch.tensor([1.0625, 1.1875, 1.3125, 2.125, 17.0, 19.0, 0.0048828125, 0.0009765625, 0.0029296875, -1.0625, 0.0, 448.0])
    x = torch.stack([torch.cat([steps, torch.zeros(116)]) * 2.0 ** p for p in (-100, -7, 0, 9, 100)])
    x = torch.cat([x, x.clone(), torch.full((1, 128), 2.0 ** -149), torch.full((1, 128), 3.0e38)])
    x[5:10, 11] *= 1.0 + 2.0 ** -23
    assert torch.equal(k.from_float8(k.to_float8(x.to(DEVICE))).double().cpu(), plain.rows(x))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [3, 40, 150])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_a_value_that_is_not_finite_makes_its_row_nan_and_no_other(k, bad, dtype, n, out_dtype):
    x, (w, held) = _rows(n, 300, dtype, 1), _weight(k, 1, 50, 300, 2)
    whole = torch.empty((n, 50), dtype=out_dtype, device=DEVICE)
    k.gemm(x.to(DEVICE), w, whole)
    x[1, 290] = bad
    out = torch.empty_like(whole)
    k.gemm(x.to(DEVICE), w, out)
    assert bool(torch.isnan(out[1]).all())
    keep = [i for i in range(n) if i != 1]
    assert torch.equal(out[keep], whole[keep])


@pytest.mark.parametrize("gate", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,width", [(3, 70), (33, 512), (20, 1001)])
def test_gated_rows_in_8_bits(k, gate, dtype, n, width):
    x = _rows(n, 2 * width, dtype, 5)
    g, u = x[:, :width].double(), x[:, width:].double()
    act = g * torch.sigmoid(g) if gate == "silu" else 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)))
    value = act * u
    held, off = plain.requantised(value, value.abs() * 2.0 ** -15 + 1e-37)
    got = k.from_float8(k.to_float8(x.to(DEVICE), gate=gate)).double().cpu()
    assert bool(((got - held).abs() <= off).all())
    assert (got != held).double().mean() < 0.01      # only what lies next to a border may fall on its other side


@pytest.mark.parametrize("weight_dtype", [torch.float32, torch.bfloat16, None])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,width", [(17, 1), (33, 70), (40, 512), (130, 1001), (300, 4096), (18, 8192)])
def test_normed_rows_in_8_bits(k, weight_dtype, dtype, n, width):
    """float32 sums of squares of up to 8192 values in 8 + 6 + 16 roundings, half of their 2^-24 each in the root, and five more: 20 * 2^-24 of a value.
    Rounded to bfloat16 on the way, that may give its neighbour, 2^-7 of it away."""
    x = _rows(n, width, torch.float32, 5) * 3.0
    x[1] = 0.0
    weight = None if weight_dtype is None else (torch.randn(width, generator=torch.Generator().manual_seed(2)) + 1.0).to(weight_dtype)
    value = x.double() / torch.sqrt((x.double() ** 2).mean(dim=1, keepdim=True) + 1e-5) * (1.0 if weight is None else weight.double())
    on_device = x.to(DEVICE), None if weight is None else weight.to(DEVICE), 1e-5
    rows = k.rmsnorm_float8(*on_device, dtype)
    got = k.from_float8(rows).double().cpu()
    if dtype == torch.bfloat16:      # the same bytes as from the rounded norm, but for a sum of squares in another order
        rounded = torch.empty((n, width), dtype=dtype, device=DEVICE)
        k.rmsnorm(*on_device, rounded)
        value = rounded.double().cpu()
    held, off = plain.requantised(value, value.abs() * (2.0 ** -19 if dtype == torch.float32 else 2.0 ** -7) + 1e-37)
    assert bool(((got - held).abs() <= off).all())
    assert (got != held).double().mean() < 0.01      # only what lies next to a border may fall on its other side
    w, matrix = _weight(k, 1, 50, width, 3)
    out = torch.empty((n, 50), device=DEVICE)
    k.gemm(rows, w, out)
    _close(out, *plain.product(got, plain.matrix(*matrix), True))


def test_normed_rows_where_the_kernel_has_none(k):
    from beholdd.kernels.library import KernelError
    assert k.rmsnorm_float8(torch.ones((16, 64), device=DEVICE), None, 1e-5) is None
    assert k.rmsnorm_float8(torch.ones((17, 8200), device=DEVICE), None, 1e-5) is None
    for x, weight in ((torch.ones((20, 64), device=DEVICE, dtype=torch.bfloat16), None), (torch.ones((20, 64), device=DEVICE), torch.ones(63, device=DEVICE)),
                      (torch.ones(64, device=DEVICE), None), (torch.ones((20, 128), device=DEVICE)[:, ::2], None)):
        with pytest.raises(KernelError):
            k.rmsnorm_float8(x, weight, 1e-5)


@pytest.mark.parametrize("matrices,n,width", [(1, 1, 1), (1, 130, 257), (2, 24, 128), (3, 144, 300)])
def test_weights_in_8_bits(k, matrices, n, width):
    w, held = _weight(k, matrices, n, width, 3)
    assert torch.equal(w.scales.cpu(), held[1])
    assert torch.equal(k.unpack_float8(w).cpu(), (held[0].float() * plain.matrix(torch.ones_like(held[0]), held[1]).float()))
    again = k.pack_float8(held[0].float().to(torch.float8_e4m3fn).to(DEVICE), held[1].to(DEVICE))
    assert torch.equal(again.data, w.data) and torch.equal(again.scales, w.scales)


# ---- products ------------------------------------------------------------------------------------------------------

SIZES = [(1, 1, 1), (1, 16, 128), (2, 100, 5), (7, 257, 640), (16, 48, 1000), (17, 130, 129), (32, 33, 384), (33, 64, 128), (45, 300, 2048), (64, 129, 129),
         (65, 127, 1001), (129, 1000, 512), (300, 333, 777), (257, 512, 4096)]


@pytest.mark.parametrize("m,n,width", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("out_dtype,full", [(torch.float32, None), (torch.float32, False), (torch.bfloat16, None), (torch.bfloat16, True)])
def test_product(k, m, n, width, dtype, out_dtype, full):
    x, (w, held) = _rows(m, width, dtype, m + n), _weight(k, 1, n, width, width)
    out = torch.full((m, n), math.nan, dtype=out_dtype, device=DEVICE)
    k.gemm(x.to(DEVICE), w, out, full_sums=full)
    _close(out, *plain.product(plain.rows(x), plain.matrix(*held), out_dtype == torch.float32 if full is None else full))


@pytest.mark.parametrize("m,n,width", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate", ["silu", "gelu_tanh"])
def test_gated_product(k, m, n, width, dtype, out_dtype, gate):
    x, (w, held) = _rows(m, width, dtype, m + n), _weight(k, 2, n, width, width)
    out = torch.full((m, n), math.nan, dtype=out_dtype, device=DEVICE)
    k.gemm_swiglu(x.to(DEVICE), w, out, gate=gate)
    x8, whole, full = plain.rows(x), plain.matrix(*held), out_dtype == torch.float32
    (g, g_error), (u, u_error) = plain.product(x8, whole[:n], full), plain.product(x8, whole[n:], full)
    if gate == "silu":
        want, bound = plain.gated(g, g_error, u, u_error)
    else:      # the slope of the tanh form is at most 1.13
        act = 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)))
        want = act * u
        bound = 1.13 * g_error * (u.abs() + u_error) + act.abs() * u_error + want.abs() * 2.0 ** -15 + 1e-37
    _close(out, want, bound)


@pytest.mark.parametrize("m", [3, 20, 200])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_product_added_and_of_several_matrices(k, m, out_dtype):
    """Into what stands there; matrices whose rows are no whole blocks of 16 one behind the other."""
    x, (w, held) = _rows(m, 700, torch.bfloat16, 8), _weight(k, 3, 37, 700, 9)
    before = _rows(m, 111, out_dtype, 10)
    out = before.to(DEVICE)
    k.gemm(x.to(DEVICE), w, out, accumulate=True)
    want, bound = plain.product(plain.rows(x), plain.matrix(*held), out_dtype == torch.float32)
    _close(out, want + before.double(), bound + 2.0 ** -24 * (want.abs() + before.double().abs()))


@pytest.mark.parametrize("m", [5, 100])
def test_product_is_the_same_again_on_another_stream_and_in_a_capture(k, m):
    x, (w, _) = _rows(m, 1024, torch.bfloat16, 8).to(DEVICE), _weight(k, 2, 256, 1024, 9)
    out, gated_out = torch.empty((m, 512), dtype=torch.float32, device=DEVICE), torch.empty((m, 256), dtype=torch.bfloat16, device=DEVICE)

    def both():
        k.gemm(x, w, out)
        k.gemm_swiglu(x, w, gated_out)

    both()
    torch.cuda.synchronize()
    want = out.clone(), gated_out.clone()
    stream = torch.cuda.Stream()
    out.zero_(), gated_out.zero_()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        both()
    torch.cuda.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(gated_out, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for turn in range(3):
        x.mul_(-1.0)
        out.zero_(), gated_out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        captured = out.clone(), gated_out.clone()
        both()
        torch.cuda.synchronize()
        assert torch.equal(out, captured[0]) and torch.equal(gated_out, captured[1])


def test_a_chain_of_float8_rows_is_the_chain_of_its_steps(k):
    """`gemm` of rows that were brought into 8 bits ahead."""
    x, (w, _) = _rows(40, 512, torch.bfloat16, 8).to(DEVICE), _weight(k, 1, 100, 512, 9)
    a, b = torch.empty((40, 100), device=DEVICE), torch.empty((40, 100), device=DEVICE)
    k.gemm(x, w, a)
    k.gemm(k.to_float8(x), w, b)
    assert torch.equal(a, b)


# ---- router --------------------------------------------------------------------------------------------------------

ROUTES = [(1, 1, 1, 1, 1), (1, 128, 8, 8, 4), (5, 16, 4, 16, 6), (33, 160, 6, 8, 3), (7, 256, 8, 8, 4), (3, 1024, 32, 64, 40), (9, 300, 5, 3, 2), (4, 64, 8, 2, 1),
          (2, 63, 7, 7, 7), (6, 130, 2, 65 // 13, 1)]


@pytest.mark.parametrize("n,e,top,groups,keep", ROUTES)
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("corrected,renorm", [(True, True), (False, False)])
def test_route_in_groups(k, n, e, top, groups, keep, scoring, group_score, corrected, renorm):
    g = torch.Generator().manual_seed(e)
    logits = torch.round(4.0 * torch.randn((n, e), generator=g)) / 2.0      # many equal ones
    correction = torch.round(8.0 * torch.randn(e, generator=g)) / 64.0 if corrected else None
    want, want_weights = plain.route(logits, correction, top, scoring, groups, keep, group_score, renorm, 2.5)
    chosen = torch.empty((n, top), dtype=torch.int32, device=DEVICE)
    weights = torch.empty((n, top), dtype=torch.float32, device=DEVICE)
    wide = torch.full((n, e + 3), math.nan)
    wide[:, :e] = logits
    k.route_in_groups(wide.to(DEVICE), correction.to(DEVICE) if corrected else None, chosen, weights, scoring=scoring, groups=groups, keep=keep,
                      group_score=group_score, renorm=renorm, factor=2.5, experts=e)
    assert torch.equal(chosen.cpu().long(), want)
    assert bool(((weights.cpu().double() - want_weights).abs() <= want_weights.abs() * (2.0 ** -24 + 1e-12)).all())


def test_route_with_masked_and_broken_logits(k):
    """Minus infinity is a score of 0, a NaN counts as the lowest, and what is chosen are always different experts of open groups."""
    logits = torch.randn((6, 32), generator=torch.Generator().manual_seed(1))
    logits[0, 3:] = -math.inf
    logits[1] = -math.inf
    logits[2, :20] = math.nan
    logits[3] = math.nan
    logits[4] = torch.finfo(torch.float32).min
    logits[5] = torch.finfo(torch.float32).max
    chosen, weights = torch.empty((6, 6), dtype=torch.int32, device=DEVICE), torch.empty((6, 6), device=DEVICE)
    k.route_in_groups(logits.to(DEVICE), None, chosen, weights, groups=4, keep=2, renorm=False)
    want, want_weights = plain.route(logits, None, 6, "sigmoid", 4, 2, "top2", False, 1.0)
    for r in (0, 1, 4, 5):
        assert chosen[r].cpu().tolist() == want[r].tolist()
        assert torch.allclose(weights[r].cpu().double(), want_weights[r], rtol=2.0 ** -23, atol=0.0)
    for r in range(6):
        picked = chosen[r].cpu().tolist()
        assert len(set(picked)) == 6 and all(0 <= e < 32 for e in picked) and len({e // 8 for e in picked}) <= 2


# ---- experts -------------------------------------------------------------------------------------------------------

def _experts(k, n, width, ff, e, top, dtype, seed, out_of_range=False):
    g = torch.Generator().manual_seed(seed)
    up, held_up = _weight(k, 2 * e, ff, width, seed + 1)
    down, held_down = _weight(k, e, width, ff, seed + 2)
    chosen = torch.randint(-1 if out_of_range else 0, e + (2 if out_of_range else 0), (n, top), generator=g, dtype=torch.int32)      # the same twice among them
    weights = torch.rand((n, top), generator=g)
    return _rows(n, width, dtype, seed), chosen, weights, (up, down), (held_up, held_down)


EXPERTS = [(1, 128, 128, 4, 2), (1, 130, 33, 1, 1), (3, 64, 48, 8, 3), (20, 300, 129, 3, 4), (70, 257, 144, 2, 2), (150, 128, 64, 5, 4), (64, 96, 20, 70, 1), (2, 144, 100, 40, 5), (1, 256, 130, 64, 16), (1, 20, 4200, 9, 2), (4, 4300, 16, 6, 3)]


@pytest.mark.parametrize("n,width,ff,e,top", EXPERTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_experts(k, n, width, ff, e, top, dtype, out_dtype):
    x, chosen, weights, packed, held = _experts(k, n, width, ff, e, top, dtype, n + e)
    before = _rows(n, width, out_dtype, 77)
    out = before.to(DEVICE)
    k.experts_float8(x.to(DEVICE), chosen.to(DEVICE), weights.to(DEVICE), *packed, out)
    want, bound = plain.experts(x, chosen, weights, *held, full=out_dtype == torch.float32)
    _close(out, want + before.double(), bound + 2.0 ** -24 * (want.abs() + before.double().abs()))
    fresh = torch.full((n, width), math.nan, dtype=out_dtype, device=DEVICE)
    k.experts_float8(x.to(DEVICE), chosen.to(DEVICE), weights.to(DEVICE), *packed, fresh, fresh=True)
    _close(fresh, want, bound)


@pytest.mark.parametrize("n,e", [(1, 12), (4, 6), (90, 3)])
@pytest.mark.parametrize("form", ["through", "none_of_them", "weigh_input", "clamped"])
def test_forms_of_experts(k, n, e, form):
    x, chosen, weights, packed, held = _experts(k, n, 200, 136, e, 3, torch.bfloat16, 31, out_of_range=form in ("through", "none_of_them"))
    more = {"weigh_input": dict(weigh_input=True), "clamped": dict(limit=0.7, alpha=1.702, shift=1.0)}.get(form, {})
    through = _rows(n, 200, torch.bfloat16, 5) if form == "through" else None
    out = torch.full((n, 200), math.nan, device=DEVICE)
    k.experts_float8(x.to(DEVICE), chosen.to(DEVICE), weights.to(DEVICE), *packed, out, fresh=True, through=through.to(DEVICE) if through is not None else None, **more)
    _close(out, *plain.experts(x, chosen, weights, *held, through=through, **more))


@pytest.mark.parametrize("n", [2, 100])
def test_route_and_experts_in_a_capture(k, n):
    """Router and experts as a step runs them, replayed on other rows."""
    x, _, _, packed, _ = _experts(k, n, 256, 128, 8, 2, torch.bfloat16, 3)
    x = x.to(DEVICE)
    matrix = torch.randn((8, 256), device=DEVICE, dtype=torch.bfloat16, generator=torch.Generator(DEVICE).manual_seed(1)) / 16
    logits, out = torch.empty((n, 8), device=DEVICE), torch.empty((n, 256), device=DEVICE)
    chosen, weights = torch.empty((n, 2), dtype=torch.int32, device=DEVICE), torch.empty((n, 2), device=DEVICE)

    def step():
        k.gemm(x, matrix, logits)
        k.route_in_groups(logits, None, chosen, weights, groups=4, keep=2)
        k.experts_float8(x, chosen, weights, *packed, out, fresh=True)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(3):
        x.copy_(_rows(n, 256, torch.bfloat16, 50 + turn))
        graph.replay()
        torch.cuda.synchronize()
        got = chosen.clone(), weights.clone(), out.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(chosen, got[0]) and torch.equal(weights, got[1]) and torch.equal(out, got[2])


def test_a_large_call_of_few_experts_has_lists_for_all_its_pairs(k):
    """Every row names the same expert in all its choices."""
    n, top = 700, 4
    x, _, weights, packed, held = _experts(k, n, 128, 64, 3, top, torch.bfloat16, 3)
    chosen = torch.full((n, top), 2, dtype=torch.int32)
    out = torch.full((n, 128), math.nan, device=DEVICE)
    k.experts_float8(x.to(DEVICE), chosen.to(DEVICE), weights.to(DEVICE), *packed, out, fresh=True)
    pick = [0, 63, 64, 350, 699]
    want, bound = plain.experts(x[pick], chosen[pick], weights[pick], *held)
    _close(out[pick], want, bound)


def test_a_value_that_is_not_finite_reaches_its_experts_rows_alone(k):
    for n in (1, 20, 200):
        x, chosen, weights, packed, _ = _experts(k, n, 160, 64, 6, 2, torch.bfloat16, 3)
        out, whole = torch.empty((n, 160), device=DEVICE), torch.empty((n, 160), device=DEVICE)
        k.experts_float8(x.to(DEVICE), chosen.to(DEVICE), weights.to(DEVICE), *packed, whole, fresh=True)
        x[n // 2, 7] = math.nan
        k.experts_float8(x.to(DEVICE), chosen.to(DEVICE), weights.to(DEVICE), *packed, out, fresh=True)
        keep = [i for i in range(n) if i != n // 2]
        assert bool(torch.isnan(out[n // 2]).all()) and torch.equal(out[keep], whole[keep])


def test_a_rows_result_does_not_depend_on_the_rows_beside_it_but_by_rounding(k):
    """The same row alone, in a batch and in a prompt: the same 8 bits, sums in another order."""
    x, (w, held) = _rows(300, 1024, torch.bfloat16, 8), _weight(k, 1, 200, 1024, 9)
    want, bound = plain.product(plain.rows(x), plain.matrix(*held), True)
    for n in (1, 16, 17, 100, 129, 300):
        out = torch.empty((n, 200), device=DEVICE)
        k.gemm(x[:n].to(DEVICE), w, out)
        _close(out, want[:n], bound[:n], f"{n} rows")


@pytest.mark.parametrize("m,n,width,full", [(200, 512, 2048, True), (200, 512, 2048, False), (129, 100, 5000, True), (400, 64, 12288, False), (1000, 1030, 640, False),
                                            (2100, 300, 384, True), (700, 4000, 512, False)])
def test_tiles_and_parts_of_k(k, m, n, width, full):
    """Sizes that go to every tile and to K in parts, some rows of each."""
    x, (w, held) = _rows(m, width, torch.bfloat16, 1), _weight(k, 1, n, width, 2)
    out = torch.full((m, n), math.nan, device=DEVICE)
    k.gemm(x.to(DEVICE), w, out, full_sums=full)
    pick = sorted({0, 1, 63, 64, 127, 128, m // 2, m - 2, m - 1})
    _close(out[pick], *plain.product(plain.rows(x[pick]), plain.matrix(*held), full))
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("m", [3, 20, 70, 300])
def test_several_matrices_side_by_side(k, m):
    """A plain product with a weight of three matrices: their outputs behind one another in each row, added to what is there."""
    x, (w, held) = _rows(m, 300, torch.bfloat16, 1), _weight(k, 3, 50, 300, 2)
    before = torch.randn((m, 150), generator=torch.Generator().manual_seed(3))
    out = before.to(DEVICE)
    k.gemm(x.to(DEVICE), w, out, accumulate=True)
    want, bound = plain.product(plain.rows(x), plain.matrix(*held), True)
    _close(out, want + before.double(), bound + (want.abs() + before.abs().double()) * 2.0 ** -24)


@pytest.mark.parametrize("m,n,width,full,gated", [
    (20, 130, 640, False, False), (20, 130, 640, True, True), (48, 130, 384, True, False), (60, 130, 384, False, False), (60, 100, 384, True, True),
    (90, 130, 384, False, False), (90, 130, 384, True, True), (128, 130, 384, True, False), (100, 2050, 640, False, False), (100, 130, 3000, False, False),
    (50, 300, 5000, True, False), (129, 64, 130, False, True), (129, 64, 3000, True, True), (129, 64, 3000, False, False), (5000, 300, 130, False, False),
    (2600, 300, 130, True, True), (400, 512, 4200, False, False), (2100, 100, 3000, True, True), (1000, 2050, 4200, False, False), (400, 4100, 130, False, True),
    (2600, 300, 4200, True, True), (2100, 2050, 3000, True, False), (1000, 2050, 3000, True, True), (1000, 4100, 130, False, False), (1000, 2050, 130, True, True),
    (1000, 4100, 1500, False, False), (1000, 2050, 1500, False, True), (5000, 1030, 2048, True, False), (2100, 4100, 1000, False, False), (1000, 4100, 1000, False, True)])
def test_every_kernel_of_products_from_rows_in_8_bits(k, m, n, width, full, gated):
    """Few rows in every number of blocks, every tile of the rings, K whole and in parts, plain and gated: some rows of each."""
    matrices = 2 if gated else 1
    x, (w, held) = _rows(m, width, torch.bfloat16, 1), _weight(k, matrices, n, width, 2)
    out = torch.full((m, n), math.nan, device=DEVICE)
    (k.gemm_swiglu if gated else k.gemm)(x.to(DEVICE), w, out, full_sums=full)
    pick = sorted({0, 1, 15, 16, 31 % m, 32 % m, 63 % m, 64 % m, 127 % m, 128 % m, m // 2, m - 2, m - 1})
    x8, whole = plain.rows(x[pick]), plain.matrix(*held)
    if gated:
        want, bound = plain.gated(*plain.product(x8, whole[:n], full), *plain.product(x8, whole[n:], full))
    else:
        want, bound = plain.product(x8, whole, full)
    _close(out[pick], want, bound)
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("m,n,width", [(400, 4100, 130), (130, 700, 300), (700, 12288, 512), (2100, 6000, 384), (1000, 4100, 1000), (5000, 300, 130)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate", ["silu", "gelu_tanh"])
def test_gated_products_that_leave_rows_in_8_bits(k, m, n, width, dtype, gate):
    """The bytes of `gemm_swiglu` and `to_float8` behind it where both add up in the same order, which within a step they do; else what lies at a
    border falls on its other side.  And rows in 8 bits are read by the next product."""
    x, (w, _) = _rows(m, width, torch.bfloat16, 3).to(DEVICE), _weight(k, 2, n, width, 4)
    got = k.gemm_swiglu_float8(x, w, gate=gate, dtype=dtype)
    plainly = torch.empty((m, n), dtype=dtype, device=DEVICE)
    k.gemm_swiglu(x, w, plainly, gate=gate)
    want = k.to_float8(plainly)
    assert (got is not None) == bool(k.lib.bh_gemm_float8_gives_8(m, n, width, int(dtype == torch.float32)))
    if got is None:
        return
    a, b = k.from_float8(got), k.from_float8(want)
    assert bool(torch.isfinite(a).all()) and (a != b).double().mean().item() < 0.01
    # a step of e4m3 is 2^-3 of a value at most, and values below the smallest normal number of their stretch lie 2^-9 * 2^e apart
    least = torch.ldexp(torch.ones((), device=DEVICE), torch.frexp(plainly.float().abs().amax(dim=1, keepdim=True))[1] - 8 - 9 + 1)
    assert bool(((a - b).abs() <= torch.maximum(b.abs() * 0.1251, least)).all())
    v, _ = _weight(k, 1, 64, n, 5)
    first, second = torch.empty((m, 64), device=DEVICE), torch.empty((m, 64), device=DEVICE)
    k.gemm(got, v, first)
    k.gemm(want, v, second)
    assert float((first - second).norm() / second.norm()) < 0.0126      # 1 % of the values a step of 2^-3 off


def test_gated_products_that_do_not_leave_rows_in_8_bits(k):
    from beholdd.kernels.library import KernelError
    w = _weight(k, 2, 64, 128, 4)[0]
    assert k.gemm_swiglu_float8(torch.ones((4, 128), device=DEVICE), w) is None
    for call in (lambda: k.gemm_swiglu_float8(torch.ones((400, 64), device=DEVICE), w), lambda: k.gemm_swiglu_float8(torch.ones((400, 128), device=DEVICE), _weight(k, 1, 64, 128, 4)[0]),
                 lambda: k.gemm_swiglu_float8(torch.ones((400, 128), device=DEVICE), w, dtype=torch.float16)):
        with pytest.raises(KernelError):
            call()


# ---- refusals ------------------------------------------------------------------------------------------------------

def test_refusals(k):
    from beholdd.kernels.library import KernelError
    w, _ = _weight(k, 2, 32, 128, 1)
    x = torch.zeros((4, 128), device=DEVICE)
    out = torch.zeros((4, 64), device=DEVICE)
    refused = [
        lambda: k.gemm(x[:, :64], w, out), lambda: k.gemm(x, w, out[:, :32]), lambda: k.gemm(x.half(), w, out), lambda: k.gemm(x.t().contiguous().t(), w, out),
        lambda: k.gemm(x, w, out.half()), lambda: k.gemm(x.cpu(), w, out), lambda: k.gemm_swiglu(x, w, out),
        lambda: k.gemm_swiglu(x, _weight(k, 1, 32, 128, 1)[0], out[:, :16].contiguous()),
        lambda: k.gemm(k.to_float8(x, in_rows=True), w, out), lambda: k.gemm(x[:0], w, out[:0]), lambda: k.to_float8(x.half()), lambda: k.to_float8(x[0]),
        lambda: k.to_float8(x[:, :127].contiguous(), gate="silu"), lambda: k.to_float8(x, gate="relu"), lambda: k.to_float8(x[:, ::2]),
        lambda: k.pack_float8(x.half()), lambda: k.pack_float8(x, matrices=3), lambda: k.pack_float8(x.cpu()), lambda: k.pack_float8(x * math.inf),
        lambda: k.pack_float8(x.to(torch.float8_e4m3fn)), lambda: k.pack_float8(x.to(torch.float8_e4m3fn), torch.ones((1, 1, 2), device=DEVICE)),
        lambda: k.pack_float8(x.to(torch.float8_e4m3fn), torch.full((1, 1, 1), math.nan, device=DEVICE)), lambda: k.pack_float8(x[:0]),
    ]
    from beholdd.kernels.library import Float8Rows, Float8Weight
    refused += [lambda: Float8Weight(w.data[:-16], w.scales, 2, 32, 128), lambda: Float8Weight(w.data, w.scales[:, :, :0], 2, 32, 128),
                lambda: Float8Weight(w.data, w.scales, 2, 48, 128), lambda: Float8Rows(w.data[:16], torch.zeros((1, 16), dtype=torch.int32, device=DEVICE), 4, 128),
                lambda: k.gemm(x, Float8Weight(w.data.cpu(), w.scales.cpu(), 2, 32, 128), out)]
    logits, chosen, weights = torch.zeros((2, 16), device=DEVICE), torch.zeros((2, 4), dtype=torch.int32, device=DEVICE), torch.zeros((2, 4), device=DEVICE)
    for more in (dict(groups=3), dict(groups=0), dict(groups=4, keep=0), dict(groups=4, keep=5), dict(groups=8, keep=1), dict(scoring="tanh"),
                 dict(group_score="sum"), dict(experts=17), dict(experts=0)):
        refused.append(lambda more=more: k.route_in_groups(logits, None, chosen, weights, **more))
    refused.append(lambda: k.route_in_groups(logits, torch.zeros(15, device=DEVICE), chosen, weights))
    refused.append(lambda: k.route_in_groups(logits, None, chosen.long(), weights))
    refused.append(lambda: k.route_in_groups(logits, None, chosen, weights[:, :3].contiguous()))
    up, down = _weight(k, 4, 32, 128, 1)[0], _weight(k, 2, 128, 32, 1)[0]
    chosen, weights, out = torch.zeros((4, 2), dtype=torch.int32, device=DEVICE), torch.zeros((4, 2), device=DEVICE), torch.zeros((4, 128), device=DEVICE)
    refused += [
        lambda: k.experts_float8(x, chosen[:3], weights, up, down, out), lambda: k.experts_float8(x, chosen, weights[:, :1].contiguous(), up, down, out),
        lambda: k.experts_float8(x, chosen, weights, down, up, out), lambda: k.experts_float8(x, chosen, weights, up, down, out[:, :64]),
        lambda: k.experts_float8(x, chosen.long(), weights, up, down, out), lambda: k.experts_float8(x, chosen, None, up, down, out, weigh_input=True),
        lambda: k.experts_float8(x, chosen, weights, up, down, out, through=out[:, :3]), lambda: k.experts_float8(x.half(), chosen, weights, up, down, out),
        lambda: k.experts_float8(x, chosen, weights, up, down, out, through=x, weigh_input=True),
    ]
    for number, call in enumerate(refused):
        with pytest.raises(KernelError):
            call()
            pytest.fail(f"call {number} was not refused")
