"""Rotary positions and attention over a paged cache from their definitions in float64, and how far a kernel may be off."""
import math

import torch


def rotate(x, positions, frequencies, layout, amplitude=1.0, inverse=False):
    """x [tokens, heads, d]; the angles of far positions in float64 too (2^-53 of 10^6 radians is nothing here)."""
    y, n = x.double().clone(), len(frequencies)
    t = positions.double()[:, None] * frequencies.to(x.device)[None] * (-1 if inverse else 1)
    cos, sin = amplitude * t.cos()[:, None], amplitude * t.sin()[:, None]
    a, b = (x[..., :n], x[..., n:2 * n]) if layout == "half" else (x[..., 0:2 * n:2], x[..., 1:2 * n:2])
    a, b = a.double(), b.double()
    u, v = a * cos - b * sin, a * sin + b * cos
    if layout == "half":
        y[..., :n], y[..., n:2 * n] = u, v
    else:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = u, v
    return y


def rotate_tolerance(x, n, layout, amplitude):
    """Half a step of the result's type, and in 32 bits: cos and sin off by 4 steps and the angle by 2^-33 + 2^-25 of half a turn
    (its rounding to 24 bits), 2.0e-7 together at most, then two products and a sum: 5 half steps of |a| + |b| in all, and as much again."""
    big = x.double().abs()
    a, b = (big[..., :n], big[..., n:2 * n]) if layout == "half" else (big[..., 0:2 * n:2], big[..., 1:2 * n:2])
    s = (a + b) * abs(amplitude)
    pair = torch.cat((s, s), -1) if layout == "half" else torch.stack((s, s), -1).flatten(-2)
    tol = torch.zeros_like(big)
    tol[..., :2 * n] = pair * (torch.finfo(x.dtype).eps / 2 + 10 * 2.0 ** -24 + 4 * 2.0 ** -23)
    return tol + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps


def gather(cache, pages, length):
    """[length, heads, d] of a cache's keys or values; zeros from what is no page of it."""
    size = cache.shape[1]
    length = min(length, pages.shape[0] * size)
    at = torch.arange(length, device=cache.device)
    page = pages.to(cache.device).long()[at // size]
    bad = (page < 0) | (page >= cache.shape[0])
    got = cache[page.clamp(0, cache.shape[0] - 1), at % size]
    return torch.where(bad[:, None, None], torch.zeros_like(got), got)


def attention(q, keys, values, pages, lengths, starts=None, causal=True, scale=None, prefix=None, prefix_length=0):
    """(out, tolerance of out, lse, tolerance of lse) in float64, NaN in the rows behind the last sequence.

    tolerance: half a step of out; half a step of each weight p, which may be held in the type for the product with the values (of what
    lies below fp16's normal numbers 2^-25 of the largest weight or more); the scores' errors (d products summed in 32 bits, the scale, the
    exponent's argument) and the sums' over the keys, n 2^-24."""
    tokens, heads, d = q.shape
    group, scale = heads // keys.shape[2], d ** -0.5 if scale is None else scale
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    tol, lse, lse_tol = out.clone(), out[..., 0].clone(), out[..., 0].clone()
    step = torch.finfo(q.dtype).eps / 2
    starts = list(range(len(lengths) + 1)) if starts is None else starts
    for b, length in enumerate(lengths):
        first, last = starts[b], starts[b + 1]
        if first == last:
            continue
        k, v = gather(keys, pages[b], length).double(), gather(values, pages[b], length).double()
        seen = torch.ones(last - first, k.shape[0], dtype=torch.bool, device=q.device)
        if causal:
            seen = torch.arange(k.shape[0], device=q.device)[None] <= torch.arange(length - (last - first), length, device=q.device)[:, None]
        if prefix_length:
            k = torch.cat((gather(keys, prefix, prefix_length).double(), k))
            v = torch.cat((gather(values, prefix, prefix_length).double(), v))
            seen = torch.cat((torch.ones(last - first, prefix_length, dtype=torch.bool, device=q.device), seen), 1)
        for h in range(heads):
            kh, vh, x = k[:, h // group], v[:, h // group], q[first:last, h].double()
            s = torch.where(seen, x @ kh.t() * scale, -math.inf)
            most = s.amax(1, keepdim=True) if s.shape[1] else torch.full((last - first, 1), -math.inf, dtype=torch.float64, device=q.device)
            most = torch.where(most == -math.inf, 0.0, most)
            p = torch.where(seen, torch.exp(s - most), 0.0)
            total = p.sum(1, keepdim=True)
            # (a value that no token of the chunk sees, or not this one, takes no part, whatever it is)
            clean = torch.where(torch.isfinite(vh), vh, 0.0)
            o = torch.where(total > 0, p @ clean / total.clamp(min=1e-300), 0.0)
            for j in torch.nonzero(~torch.isfinite(vh).all(1)).flatten().tolist():
                o = o + torch.where(seen[:, j, None], torch.where(torch.isfinite(vh[j]), 0.0, vh[j]), 0.0)
            weight = torch.where(total > 0, p @ clean.abs() / total.clamp(min=1e-300), 0.0)
            parts = torch.where(seen, x.abs() @ torch.nan_to_num(kh).abs().t(), 0.0) * scale
            most_part = parts.amax(1, keepdim=True) if parts.shape[1] else torch.zeros_like(most)
            score = (d + 4) * 2.0 ** -24 * most_part + 2.0 ** -22 * most_part + s.shape[1] * 2.0 ** -24 + 2.0 ** -21
            t = step * (o.abs() + weight) + 2 * weight * score
            if q.dtype == torch.float16:
                t = t + 2.0 ** -24 * clean.abs().sum(0, keepdim=True) + 2.0 ** -25
            out[first:last, h], tol[first:last, h] = o, t + 1e-30
            lse[first:last, h] = torch.where(total > 0, most + total.clamp(min=1e-300).log(), -math.inf)[:, 0]
            lse_tol[first:last, h] = (score + 2.0 ** -22 * lse[first:last, h, None].abs().nan_to_num(0, 0, 0))[:, 0]
    return out, tol, lse, lse_tol


def compare(got, want, tol):
    """The largest error in tolerances, and whether the infinities and NaNs are those that are wanted."""
    got = got.double()
    finite = torch.isfinite(want)
    same = torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    return same, float(((got - want).abs()[finite] / tol[finite]).max()) if finite.any() else 0.0
