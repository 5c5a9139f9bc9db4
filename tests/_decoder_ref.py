"""Rotary positions, paged append and attention over a paged cache in plain float64 on the CPU, with error bounds.

The bounds follow from the arithmetic: a sum of n products in float32 is off by at most n 2^-24 times the sum of their
magnitudes (any order), a rounding to a type by half its step, and a relative error d of a score's exponent argument by a
factor e^d of its weight.
"""
import math

import torch

HALF_STEP = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def turn(x, positions, freq, interleaved=False, magnitude=1.0, inverse=False):
    """``x [B, L, H, D]`` (float64), ``positions [B, L]``; also the magnitudes |a| + |b| that a rotated channel is made of."""
    n = freq.numel()
    angle = positions.double()[:, :, None, None] * freq.double()
    cos, sin = torch.cos(angle) * magnitude, torch.sin(angle) * magnitude
    if inverse:
        sin = -sin
    y, size = x.clone(), torch.zeros_like(x)
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * magnitude
    return y, size


def turn_bound(y, size, dtype, positions, freq):
    """Cosine and sine are within two units of the last place of one (argument in turns rounded to the arithmetic's
    precision: pi half-steps; the function itself: one more), two products and a sum round three times; the angle is off by
    three roundings of float64 (frequency in turns, product, and the reduction's difference)."""
    unit = 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24
    far = float((positions.double().abs().max() * freq.double().abs().max()).item()) if positions.numel() else 0.0
    return size * (8 * unit + 3 * far * 2.0 ** -53) + HALF_STEP[dtype] * y.abs() + 1e-300 + (2.0 ** -25 if dtype == torch.float16 else 0)


def new_positions(lens, new, length):
    return (lens - new)[:, None] + torch.arange(length)


def attend(q, k_cache, v_cache, table, lens, new, kernel=None, dilation=1, scale=None):
    """Everything float64 / int64 on the CPU.  ``(out, lse, out_bound(dtype), lse_bound)``; keys on pages that are not there
    are not seen."""
    B, L, Hq, D = q.shape
    pages, ps, Hkv, _ = k_cache.shape
    group, scale = Hq // Hkv, D ** -0.5 if scale is None else scale
    out, lse = torch.zeros(B, L, Hq, D, dtype=torch.float64), torch.full((B, L, Hq), -math.inf, dtype=torch.float64)
    spread, slack = torch.zeros_like(out), torch.zeros(B, L, Hq, dtype=torch.float64)      # sum p |v|; error of a score
    count = torch.ones(B, L, Hq, dtype=torch.float64)
    for b in range(B):
        fresh = min(max(int(new[b]), 0), L)
        for i in range(fresh):
            p = max(int(lens[b]), 0) - fresh + i
            back = range(p + 1) if kernel is None else range(kernel)
            where = []
            for t in back:
                j = p - t * dilation
                if j < 0:
                    break
                n = j // ps
                if n < table.shape[1] and 0 <= int(table[b, n]) < pages:
                    where.append((int(table[b, n]), j % ps))
            if not where:
                continue
            at = torch.tensor(where)
            keys, values = k_cache[at[:, 0], at[:, 1]], v_cache[at[:, 0], at[:, 1]]        # [n, Hkv, D]
            for h in range(Hq):
                s = keys[:, h // group] @ q[b, i, h] * scale
                w = torch.softmax(s, 0)
                out[b, i, h] = w @ values[:, h // group]
                lse[b, i, h] = torch.logsumexp(s, 0)
                spread[b, i, h] = w @ values[:, h // group].abs()
                size = (keys[:, h // group].abs() @ q[b, i, h].abs()).max() * abs(scale)
                slack[b, i, h] = (D + 4) * 2.0 ** -24 * size + 2.0 ** -22
                count[b, i, h] = len(where)

    def bound(dtype):
        # weights: score and exponential (slack, twice: in the sum and in the divisor), their rounding to 16 bits before the
        # product (float32: none to speak of), and the sums themselves
        weights = HALF_STEP[dtype] + 2 * slack + 2 * count * 2.0 ** -24
        # a weight below float16's smallest normal number is rounded to half a step of 2^-24 (times the largest weight, 1)
        tiny = (count * 2.0 ** -25)[..., None] * float(v_cache.nan_to_num().abs().max() if v_cache.numel() else 0) if dtype == torch.float16 else 0
        return spread * weights[..., None] + HALF_STEP[dtype] * out.abs() + tiny + 1e-30

    shown = torch.where(torch.isfinite(lse), lse.abs(), 0)
    return out, lse, bound, slack + count * 2.0 ** -24 + (shown + 8) * 2.0 ** -22


def check(name, got, want, bound):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    finite = torch.isfinite(want)
    assert torch.equal(finite, torch.isfinite(got)), f"{name}: finite pattern differs"
    assert torch.allclose(want[~finite], got[~finite], equal_nan=True), f"{name}: infinities or NaN differ"
    over = ((got - want).abs() - bound)[finite]
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 0, f"{name}: {worst:.3e} over its bound, largest difference {float((got - want).abs()[finite].max()):.3e}"
