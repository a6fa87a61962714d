"""Operators of a model whose weights are kept in 8 bits, as cases whose time is worth measuring.

  product   a linear layer: rows of activations times a weight matrix in 8-bit floating point (e4m3) with a scale for each block of
            128 x 128, plain or through the gate of a gated feed-forward
  route     the router of a mixture of experts: scores, a correction of the choice for balance, groups of experts of which a row
            may use a few, the largest of what is left, weights that are normed over the chosen
  experts   the experts' gated feed-forwards for the chosen (row, expert) pairs, their matrices in 8 bits, summed by the weights

Rows go into a product in 8 bits too.  A stretch of 128 values of a row has the scale 2^e with the least e for which no value exceeds
448 * 2^e, and a value is rounded once, to the nearest e4m3 of value / 2^e (ties to even).  A product's sum over such a stretch is
multiplied by both scales, and these are added up in 32 bits.

Layer sizes are those of `bench.py` and of `perf/cases.py` (widths of 1,024 to 5,120, feed-forwards of up to 17,408) or generic.
"""

import math

import torch

own = False

DEVICE = "cuda:0"
BLOCK = 128
LARGEST = 448.0      # of e4m3


# ---- the cases ----------------------------------------------------------------------------------------------------

def listed():
    return [
        # One user's next token: queries, keys and values of a layer.  Launches and reading the matrix.
        dict(name="product_1_qkv", do="product", rows=1, inputs=4096, outputs=6144, gated=False, dtype="bfloat16", out="bfloat16"),
        # Eight users' next tokens through the widest matrix of a layer.
        dict(name="product_8_gated", do="product", rows=8, inputs=4096, outputs=12288, gated=True, dtype="bfloat16", out="bfloat16"),
        # A batch of answers, or one short question: too few rows to fill the chip; added to a 32-bit residual afterwards.
        dict(name="product_45_down", do="product", rows=45, inputs=12288, outputs=4096, gated=False, dtype="bfloat16", out="float32"),
        # A prompt of a smaller model in 32 bits, no size a multiple of anything.
        dict(name="product_777_ragged", do="product", rows=777, inputs=1000, outputs=1333, gated=False, dtype="float32", out="float32"),
        # A prompt of 2,048 tokens, the projection behind the attention.
        dict(name="product_2048_square", do="product", rows=2048, inputs=4096, outputs=4096, gated=False, dtype="bfloat16", out="bfloat16"),
        # The largest step there is in ordinary use.
        dict(name="product_8160_gated", do="product", rows=8160, inputs=4096, outputs=12288, gated=True, dtype="bfloat16", out="bfloat16"),
        # One user's next token.
        dict(name="route_1_of_128", do="route", rows=1, experts=128, top=8, groups=8, keep=4, scoring="sigmoid", group_score="top2",
             correction=True, renorm=True, factor=2.5),
        # Prompts through a large mixture.
        dict(name="route_8192_of_256", do="route", rows=8192, experts=256, top=8, groups=8, keep=4, scoring="sigmoid", group_score="top2",
             correction=True, renorm=True, factor=2.5),
        # Softmax scores, groups judged by their best expert, weights as the scores are.
        dict(name="route_1234_of_160", do="route", rows=1234, experts=160, top=6, groups=8, keep=3, scoring="softmax", group_score="max",
             correction=False, renorm=False, factor=16.0),
        # One user's next token through eight experts.
        dict(name="experts_1", do="experts", rows=1, width=2048, ff=768, experts=128, top=8, dtype="bfloat16", out="bfloat16"),
        # A server's batch: nearly every expert has a pair or two.
        dict(name="experts_64", do="experts", rows=64, width=2048, ff=768, experts=128, top=8, dtype="bfloat16", out="bfloat16"),
        # Prompts: every expert has some hundred pairs.
        dict(name="experts_4096", do="experts", rows=4096, width=4096, ff=1536, experts=32, top=4, dtype="bfloat16", out="bfloat16"),
    ]


def _between(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _width(rng, low, high):
    """The width of a layer: most are multiples of 128, some of 16, some of nothing."""
    width = _between(rng, low, high)
    kind = rng.choice([128, 128, 128, 16, 1])
    return max(low, width // kind * kind)


def draw(rng):
    do = rng.choice(["product", "product", "route", "experts"])
    if do == "product":
        gated = rng.random() < 0.4
        case = dict(do=do, rows=_between(rng, 1, 8160), inputs=_width(rng, 512, 12288), outputs=_width(rng, 512, 12288), gated=gated,
                    dtype=rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"]), out="bfloat16" if gated else rng.choice(["bfloat16", "float32"]))
        most = 8160 * 4096 * 2 * 12288      # the largest listed case's
        case["rows"] = min(case["rows"], most // (case["inputs"] * case["outputs"] * (2 if gated else 1)))
        return case
    if do == "route":
        groups = rng.choice([1, 2, 4, 8, 8])
        experts = groups * rng.randint(max(2, 16 // groups), 256 // groups)
        keep = rng.randint(max(1, groups // 4), groups)
        scoring = rng.choice(["sigmoid", "softmax"])
        return dict(do=do, rows=_between(rng, 1, 8192), experts=experts, top=rng.randint(1, min(8, keep * (experts // groups))), groups=groups,
                    keep=keep, scoring=scoring, group_score=rng.choice(["top2", "max"]), correction=rng.random() < 0.6,
                    renorm=rng.random() < 0.6, factor=rng.choice([1.0, 2.5, 16.0]))
    width, ff, experts = _width(rng, 512, 4096), _width(rng, 128, 1536), _between(rng, 8, 128)
    top = rng.randint(1, 8)
    experts = max(top, min(experts, 32 * 4096 * 1536 // (width * ff)))
    return dict(do=do, rows=max(1, min(_between(rng, 1, 4096), 4096 * 4 * 4096 * 1536 // (top * width * ff))), width=width, ff=ff, experts=experts, top=top,
                dtype=rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"]), out="bfloat16")


def work(case):
    n = case["rows"]
    if case["do"] == "product":
        k, wide = case["inputs"], case["outputs"] * (2 if case["gated"] else 1)
        held = wide * k + 4 * -(-case["outputs"] // BLOCK) * (2 if case["gated"] else 1) * -(-k // BLOCK)
        return {"bytes": held + n * k * _size(case["dtype"]) + n * case["outputs"] * _size(case["out"]), "flops": 2 * n * wide * k}
    if case["do"] == "route":
        e = case["experts"]
        return {"bytes": 4 * n * e + (4 * e if case["correction"] else 0) + 8 * n * case["top"], "flops": n * e * (8 + case["top"])}
    width, ff, pairs = case["width"], case["ff"], n * case["top"]
    used = min(case["experts"], pairs)      # an expert without a pair need not be read
    return {"bytes": used * 3 * width * ff + n * width * (_size(case["dtype"]) + _size(case["out"])) + 8 * pairs, "flops": 6 * pairs * width * ff}


def _size(dtype):
    return {"bfloat16": 2, "float32": 4}[dtype]


# ---- inputs -------------------------------------------------------------------------------------------------------

_kernels = None


def _library():
    """The framework's kernels, loaded once for the process as an engine does."""
    global _kernels
    if _kernels is None:
        from beholdd.kernels import HipKernels

        _kernels = HipKernels(DEVICE)
    return _kernels


def _normal(shape, generator):
    return torch.randn(shape, generator=generator, device=DEVICE, dtype=torch.float32)


def _activations(rows, width, dtype, generator):
    """What stands behind a norm: about 1, some channels ten and more times as large, another level for each row."""
    channels = 1.0 + 15.0 * (torch.rand(width, generator=generator, device=DEVICE) < 0.01) * torch.rand(width, generator=generator, device=DEVICE)
    level = torch.exp(0.5 * _normal((rows, 1), generator))
    return (_normal((rows, width), generator) * channels * level).to(getattr(torch, dtype))


def _blocks(count):
    return -(-count // BLOCK)


def _weight(matrices, rows, width, generator):
    """(values [matrices * rows, width] in e4m3, scales [matrices, blocks of rows, blocks of columns]) as a checkpoint in 8 bits holds
    them: in each block the largest of the values stands at the largest that e4m3 holds."""
    values = torch.empty((matrices, rows, width), dtype=torch.float8_e4m3fn, device=DEVICE)
    scales = torch.empty((matrices, _blocks(rows), _blocks(width)), dtype=torch.float32, device=DEVICE)
    for m in range(matrices):
        w = torch.zeros((_blocks(rows) * BLOCK, _blocks(width) * BLOCK), device=DEVICE)
        w[:rows, :width] = _normal((rows, width), generator) / math.sqrt(width)
        tiles = w.view(_blocks(rows), BLOCK, _blocks(width), BLOCK)
        scales[m] = tiles.abs().amax(dim=(1, 3)) / LARGEST
        values[m] = (tiles / scales[m][:, None, :, None]).view(w.shape)[:rows, :width].to(torch.float8_e4m3fn)
    return values.view(matrices * rows, width), scales


def _inputs(case, seed):
    generator = torch.Generator(device=DEVICE).manual_seed(int(seed) % (1 << 62))
    if case["do"] == "product":
        x = _activations(case["rows"], case["inputs"], case["dtype"], generator)
        return dict(x=x, w=_weight(2 if case["gated"] else 1, case["outputs"], case["inputs"], generator))
    if case["do"] == "route":
        made = dict(logits=2.0 * _normal((case["rows"], case["experts"]), generator), correction=None)
        if case["correction"]:
            made["correction"] = 0.1 * _normal((case["experts"],), generator)
        return made
    n, e, top = case["rows"], case["experts"], case["top"]
    liking = _normal((n, e), generator) + 0.5 * _normal((1, e), generator)      # some experts are asked more often
    picked = liking.topk(top, dim=1)
    return dict(x=_activations(n, case["width"], case["dtype"], generator), chosen=picked.indices.to(torch.int32).contiguous(),
                weights=torch.softmax(picked.values, dim=1).contiguous(), up=_weight(2 * e, case["ff"], case["width"], generator),
                down=_weight(e, case["width"], case["ff"], generator))


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    if own:
        k = state["kernels"] = _library()
        for name in ("w", "up", "down"):
            if name in state:
                state[name] = k.pack_float8(*state[name])
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    case, k = state["case"], state["kernels"]
    if case["do"] == "product":
        out = torch.empty((case["rows"], case["outputs"]), dtype=getattr(torch, case["out"]), device=DEVICE)
        (k.gemm_swiglu if case["gated"] else k.gemm)(state["x"], state["w"], out)
        return out
    if case["do"] == "route":
        chosen = torch.empty((case["rows"], case["top"]), dtype=torch.int32, device=DEVICE)
        weights = torch.empty((case["rows"], case["top"]), dtype=torch.float32, device=DEVICE)
        k.route_in_groups(state["logits"], state["correction"], chosen, weights, scoring=case["scoring"], groups=case["groups"], keep=case["keep"],
                          group_score=case["group_score"], renorm=case["renorm"], factor=case["factor"])
        return chosen, weights
    out = torch.empty((case["rows"], case["width"]), dtype=getattr(torch, case["out"]), device=DEVICE)
    k.experts_float8(state["x"], state["chosen"], state["weights"], state["up"], state["down"], out, fresh=True)
    return out


def _in_8_bits(x):
    """Rows as a product takes them: (values of e4m3 in 32 bits, a scale for each value), 32-bit arithmetic whose steps are exact."""
    n, width = x.shape
    padded = torch.zeros((n, _blocks(width) * BLOCK), dtype=torch.float32, device=x.device)
    padded[:, :width] = x
    padded = padded.view(n, _blocks(width), BLOCK)
    mantissa, exponent = torch.frexp(padded.abs().amax(dim=2, keepdim=True))      # largest = mantissa * 2^exponent, mantissa in [0.5, 1)
    exponent = (exponent - 9 + (mantissa > LARGEST / 512).to(exponent.dtype)).clamp(min=-126)
    scale = torch.ldexp(torch.ones_like(mantissa), exponent)
    return (padded / scale).to(torch.float8_e4m3fn).to(torch.float32), scale


def _times(x, values, scales):
    """x [n, K] times values [N, K]^T with a scale for each block of 128 x 128."""
    quantised, scale = _in_8_bits(x)
    rows = (quantised * scale).view(x.shape[0], -1)[:, :x.shape[1]]
    spread = scales.repeat_interleave(BLOCK, dim=0).repeat_interleave(BLOCK, dim=1)
    return rows @ (values.to(torch.float32) * spread[:values.shape[0], :values.shape[1]]).t()


def _gated(x, values, scales):
    half = values.shape[0] // 2
    gate, up = _times(x, values[:half], scales[0]), _times(x, values[half:], scales[1])
    return gate / (1.0 + torch.exp(-gate)) * up


def _run_plain(state):
    case = state["case"]
    if case["do"] == "product":
        values, scales = state["w"]
        out = _gated(state["x"], values, scales) if case["gated"] else _times(state["x"], values, scales[0])
        return out.to(getattr(torch, case["out"]))
    if case["do"] == "route":
        return _route_plain(state)
    x, chosen, weights = state["x"], state["chosen"], state["weights"]
    out = torch.zeros((case["rows"], case["width"]), dtype=torch.float32, device=DEVICE)
    ff, width = case["ff"], case["width"]
    for e in range(case["experts"]):
        row, choice = torch.nonzero(chosen == e, as_tuple=True)
        if row.numel():
            inner = _gated(x[row].to(torch.float32), state["up"][0][2 * e * ff:2 * (e + 1) * ff], state["up"][1][2 * e:2 * e + 2])
            share = _times(inner, state["down"][0][e * width:(e + 1) * width], state["down"][1][e])
            out.index_add_(0, row, share * weights[row, choice][:, None])
    return out.to(getattr(torch, case["out"]))


def _route_plain(state):
    case = state["case"]
    z = state["logits"].to(torch.float64)      # two scores may lie closer than 32 bits tell apart
    n, e = z.shape
    if case["scoring"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-z))
    else:
        score = torch.exp(z - z.amax(dim=1, keepdim=True))
        score = score / score.sum(dim=1, keepdim=True)
    by = score if state["correction"] is None else score + state["correction"].to(torch.float64)
    if case["keep"] < case["groups"]:
        each = e // case["groups"]
        grouped = by.view(n, case["groups"], each)
        if case["group_score"] == "max" or each == 1:
            merit = grouped.amax(dim=2)
        else:
            ordered = torch.sort(grouped, dim=2, descending=True).values
            merit = ordered[:, :, 0] + ordered[:, :, 1]
        kept = torch.sort(merit, dim=1, descending=True, stable=True).indices[:, :case["keep"]]
        open_groups = torch.zeros_like(merit, dtype=torch.bool).scatter_(1, kept, True)
        by = torch.where(open_groups.repeat_interleave(each, dim=1), by, torch.full_like(by, -math.inf))
    chosen = torch.sort(by, dim=1, descending=True, stable=True).indices[:, :case["top"]]
    weights = torch.gather(score, 1, chosen)
    if case["renorm"]:
        weights = weights / weights.sum(dim=1, keepdim=True)
    return chosen.to(torch.int32), (weights * case["factor"]).to(torch.float32)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _exact_rows(x):
    """The values that rows stand for in 8 bits, from their definition."""
    n, width = x.shape
    held = torch.empty((n, width), dtype=torch.float64, device=x.device)
    for first in range(0, width, BLOCK):
        part = x[:, first:first + BLOCK].to(torch.float64)
        largest = part.abs().max(dim=1, keepdim=True).values
        e = torch.full_like(largest, -126.0)
        positive = largest > 0
        guess = torch.floor(torch.log2(torch.where(positive, largest, torch.ones_like(largest)) / LARGEST)) - 1.0
        for _ in range(3):
            guess = torch.where(LARGEST * torch.exp2(guess) < largest, guess + 1.0, guess)
        e = torch.where(positive, torch.maximum(guess, e), e)
        v = part / torch.exp2(e)
        step = torch.exp2(torch.clamp(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -20))), min=-6.0) - 3.0)
        held[:, first:first + BLOCK] = torch.round(v / step) * step * torch.exp2(e)
    return held


def _exact_matrix(values, scales):
    w = values.to(torch.float32).to(torch.float64)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            w[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= scales[i, j].to(torch.float64)
    return w


def _exact_gated(rows, values, scales):
    half = values.shape[0] // 2
    gate = torch.matmul(rows, _exact_matrix(values[:half], scales[0]).t())
    return gate * torch.sigmoid(gate) * torch.matmul(rows, _exact_matrix(values[half:], scales[1]).t())


def _exact_route(case, made):
    import numpy as np

    z = made["logits"].cpu().numpy().astype(np.float64)
    correction = made["correction"].cpu().numpy().astype(np.float64) if made["correction"] is not None else np.zeros(z.shape[1])
    each = case["experts"] // case["groups"]
    chosen = np.empty((z.shape[0], case["top"]), dtype=np.int32)
    weights = np.empty((z.shape[0], case["top"]))
    for r, row in enumerate(z):
        score = 1.0 / (1.0 + np.exp(-row)) if case["scoring"] == "sigmoid" else np.exp(row - row.max()) / np.exp(row - row.max()).sum()
        by = score + correction
        allowed = list(range(case["experts"]))
        if case["keep"] < case["groups"]:
            merits = []
            for g in range(case["groups"]):
                best = sorted(by[g * each:(g + 1) * each], reverse=True)[:2 if case["group_score"] == "top2" else 1]
                merits.append((-sum(best), g))
            groups = {g for _, g in sorted(merits)[:case["keep"]]}
            allowed = [i for i in allowed if i // each in groups]
        best = sorted(allowed, key=lambda i: (-by[i], i))[:case["top"]]
        chosen[r] = best
        weights[r] = score[best] / (score[best].sum() if case["renorm"] else 1.0) * case["factor"]
    return torch.from_numpy(chosen), torch.from_numpy(weights)


def exact(case, seed):
    made = _inputs(case, seed)
    if case["do"] == "route":
        return _exact_route(case, made)
    if case["do"] == "product":
        rows, (values, scales) = _exact_rows(made["x"]), made["w"]
        if case["gated"]:
            return _exact_gated(rows, values, scales)
        return torch.matmul(rows, _exact_matrix(values, scales[0]).t())
    rows, (up, up_scales), (down, down_scales) = _exact_rows(made["x"]), made["up"], made["down"]
    out = torch.zeros((case["rows"], case["width"]), dtype=torch.float64, device=DEVICE)
    ff, width = case["ff"], case["width"]
    for e in range(case["experts"]):
        for choice in range(case["top"]):
            mine = made["chosen"][:, choice] == e
            if bool(mine.any()):
                inner = _exact_gated(rows[mine], up[2 * e * ff:2 * (e + 1) * ff], up_scales[2 * e:2 * e + 2])
                share = torch.matmul(_exact_rows(inner), _exact_matrix(down[e * width:(e + 1) * width], down_scales[e]).t())
                out[mine] += share * made["weights"][mine, choice].to(torch.float64)[:, None]
    return out
