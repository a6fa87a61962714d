"""Products in 8 bits, the router in groups and experts in 8 bits in 64-bit arithmetic, from their definitions, with bounds on what 32-bit
sums in any order may differ from them by.  Everything on the CPU."""

import math

import torch

BLOCK, LARGEST = 128, 448.0
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16)}      # of a rounding, relative to the value


def e4m3(v):
    """The nearest e4m3 of values of at most 448, ties to even."""
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -30))), min=-6.0) - 3.0)
    return torch.round(v / step) * step


def exponents(x):
    """The exponent of each stretch's scale, [n, stretches]: the least e >= -126 with max |x| <= 448 * 2^e."""
    n, width = x.shape
    stretches = -(-width // BLOCK)
    padded = torch.zeros((n, stretches * BLOCK), dtype=torch.float64)
    padded[:, :width] = x.to(torch.float64)
    largest = padded.view(n, stretches, BLOCK).abs().amax(dim=2)
    e = torch.full_like(largest, -126.0)
    while bool((LARGEST * torch.exp2(e) < largest).any()):
        e = torch.where(LARGEST * torch.exp2(e) < largest, e + 1.0, e)
    return e


def rows(x):
    """What rows stand for in 8 bits."""
    scale = torch.exp2(exponents(x)).repeat_interleave(BLOCK, dim=1)[:, :x.shape[1]]
    return e4m3(x.to(torch.float64) / scale) * scale


def quantised_matrix(w, matrices=1):
    """(values, scales [matrices, ...]) of a float32 matrix as `pack_float8` makes them: the scale and the quotient are float32."""
    n = w.shape[0] // matrices
    n_blocks, k_blocks = -(-n // BLOCK), -(-w.shape[1] // BLOCK)
    values, scales = torch.empty(w.shape, dtype=torch.float64), torch.ones((matrices, n_blocks, k_blocks), dtype=torch.float32)
    for m in range(matrices):
        for i in range(n_blocks):
            for j in range(k_blocks):
                at = (slice(m * n + i * BLOCK, min(m * n + (i + 1) * BLOCK, (m + 1) * n)), slice(j * BLOCK, (j + 1) * BLOCK))
                block = w[at].to(torch.float32)
                if float(block.abs().max()) > 0:
                    scales[m, i, j] = block.abs().max() / LARGEST
                values[at] = e4m3((block / scales[m, i, j]).to(torch.float64))
    return values, scales


def matrix(values, scales):
    """The matrix that values [matrices * n, K] with scales [matrices, ...] stand for."""
    matrices, n = scales.shape[0], values.shape[0] // scales.shape[0]
    spread = scales.to(torch.float64).repeat_interleave(BLOCK, dim=1)[:, :n].repeat_interleave(BLOCK, dim=2)[:, :, :values.shape[1]]
    return values.to(torch.float64) * spread.reshape(values.shape)


def product(x8, w, full):
    """(x8 @ w^T, a bound on the error of its sums).  Full sums: the products are exact in float32, and every one of them goes through at
    most 128 additions of its stretch, the scales' product and the fused multiply-add (3), and one addition for each stretch, part and wave.
    The matrix cores' own: 8 neighbouring products are aligned to the largest, of which each loses less than 2^-13 (8 * 2^-13 of the
    largest for the eight, so 2^-10 of their magnitudes' sum), then float32 as before."""
    magnitudes = x8.abs() @ w.abs().t()
    additions = 128 + 3 + -(-x8.shape[1] // BLOCK) + 32
    return x8 @ w.t(), magnitudes * (additions * 2.0 ** -24 + (0.0 if full else 2.0 ** -10)) + 1e-37


def gated(gate, gate_error, up, up_error, limit=math.inf, alpha=1.0, shift=0.0):
    """act(gate) * (up + shift) and a bound: the slope of g sigmoid(alpha g) is at most 1.1 in magnitude, the exponential, the division and
    the products each round by 2^-24, the exponential's argument by 2^-23 of itself (at most 90 before the sigmoid is 0 or 1)."""
    g, u = gate.clamp(max=limit), up.clamp(min=-limit, max=limit)
    act = g * torch.sigmoid(alpha * g)
    value = act * (u + shift)
    return value, 1.1 * gate_error * (u + shift).abs() + act.abs() * up_error + 1.1 * gate_error * up_error + value.abs() * 2.0 ** -15 + 1e-37


def requantised(value, error):
    """(what `value` stands for in 8 bits, how far what it stands for may be off when `value` is off by up to `error`)."""
    held = rows(value)
    return held, torch.maximum((rows(value + error) - held).abs(), (rows(value - error) - held).abs())


def experts(x, chosen, weights, up, down, limit=math.inf, alpha=1.0, shift=0.0, weigh_input=False, through=None, full=True):
    """(out, bound) for up (values, scales) of 2 E matrices and down of E; `full` says how the down product sums (the up product's are full)."""
    w_up, w_down = matrix(*up), matrix(*down)
    e_count = down[1].shape[0]
    ff, width = up[0].shape[0] // (2 * e_count), down[0].shape[0] // e_count
    x8 = rows(x)
    out, bound = torch.zeros((x.shape[0], width), dtype=torch.float64), torch.zeros((x.shape[0], width), dtype=torch.float64)
    for r in range(x.shape[0]):
        for j in range(chosen.shape[1]):
            e, weight = int(chosen[r, j]), (1.0 if weights is None else float(weights[r, j]))
            if 0 <= e < e_count:
                g, g_error = product(x8[r:r + 1], w_up[2 * e * ff:(2 * e + 1) * ff], True)
                u, u_error = product(x8[r:r + 1], w_up[(2 * e + 1) * ff:(2 * e + 2) * ff], True)
                if weigh_input:
                    g, g_error, u, u_error = g * weight, abs(weight) * g_error + 2.0 ** -24 * g.abs(), u * weight, abs(weight) * u_error + 2.0 ** -24 * u.abs()
                    weight = 1.0
                inner, off = requantised(*gated(g, g_error, u, u_error, limit, alpha, shift))
                w = w_down[e * width:(e + 1) * width]
                y, y_error = product(inner, w, full)
                share, error = y[0], y_error[0] + (off @ w.abs().t())[0] * 1.01
            elif e >= e_count and through is not None:
                share, error = through[r].to(torch.float64), torch.zeros(width, dtype=torch.float64)
            else:
                continue
            out[r] += weight * share
            bound[r] += abs(weight) * (error + (chosen.shape[1] + 2) * 2.0 ** -24 * share.abs())
    return out, bound


def route(logits, correction, top, scoring, groups, keep, group_score, renorm, factor):
    """(chosen, weights) by sorting."""
    z = logits.to(torch.float64)
    score = torch.sigmoid(z) if scoring == "sigmoid" else torch.softmax(z, dim=1)
    by = score if correction is None else score + correction.to(torch.float64)
    by = torch.where(torch.isnan(by), torch.full_like(by, -math.inf), by)
    n, e = by.shape
    each, chosen = e // groups, []
    for r in range(n):
        allowed = range(e)
        if keep < groups:
            merits = []
            for g in range(groups):
                best = sorted(by[r, g * each:(g + 1) * each].tolist(), reverse=True)[:2 if group_score == "top2" else 1]
                merits.append((-sum(best), g))
            kept = {g for _, g in sorted(merits)[:keep]}
            allowed = [i for i in range(e) if i // each in kept]
        chosen.append(sorted(allowed, key=lambda i: (-float(by[r, i]), i))[:top])
    chosen = torch.tensor(chosen, dtype=torch.int64)
    weights = torch.gather(score, 1, chosen)
    if renorm:
        total = weights.sum(dim=1, keepdim=True)
        weights = torch.where(total == 0, torch.zeros_like(weights), weights / total)
    return chosen, weights * factor
