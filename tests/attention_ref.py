"""Rotary positions, the paged cache's writer and attention over it in 64 bits, each with the
largest error that fp32 arithmetic and the roundings allow.

u = 2^-24 is fp32's half step. A turned element: the angle in half turns carries a half step of at
most 1 (pi u / 2 in radians) and 2^-32 of a turn, cosine and sine two steps, the two products and their
sum three half steps of (|a| + |b|): 8 u of it in all. Frequencies are 64-bit numbers, off by 2^-53 of
themselves and as much again through 1 / 2 pi and their product with the position.

Attention: a score's D products are exact and their sum is off by D u sum |q k|, scale and exponent
two more half steps of the score and of its distance from the maximum; weights are rounded to the type
(h of each, and 2^-25 below fp16's normal range); their n sums by n u. Roundings of different weights are
independent and bounded, so that their sum passes 8 root sums of squares with a probability of 2 e^-32;
h |o| more where they agree."""
import math

import torch

from operators_ref import U, half_step


def frequencies(dim, base, scaling=None, factor=1.0, original=None, fast=32.0, slow=1.0):
    """(radians per position [dim/2] in 64 bits, factor on cosine and sine)"""
    if scaling == "base":
        base = base * factor ** (dim / (dim - 2))
    i = torch.arange(dim // 2, dtype=torch.float64)
    f = torch.tensor(base, dtype=torch.float64) ** (-2 * i / dim)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "parts":
        at = [dim * math.log(original / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (fast, slow)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dim - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1
    return f, 1.0


def rotate(x, positions, f, turn, layout):
    """(turned x [..., heads, D], bound)"""
    n = f.shape[0]
    v, f = x.double(), f.to(x.device)
    p = positions.double()[..., None, None]
    a, b = ((slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2)))
    c, s = (p * f).cos() * turn, (p * f).sin() * turn
    out, err = v.clone(), torch.zeros_like(v)
    out[..., a], out[..., b] = v[..., a] * c - v[..., b] * s, v[..., b] * c + v[..., a] * s
    off = (v[..., a].abs() + v[..., b].abs()) * abs(turn) * (8 * U + (p * f).abs() * 2.0 ** -51)
    err[..., a], err[..., b] = off, off
    bound = err + half_step(out, x.dtype)
    bound[..., 2 * n:] = 0
    return out, bound


def places(table, lengths, starts, page, pages):
    """For each sequence (first row, new rows, position of the first, [position -> flat place or -1])."""
    B, width = table.shape
    starts = list(range(B + 1)) if starts is None else starts.tolist()
    res = []
    for b in range(B):
        n, length = starts[b + 1] - starts[b], int(lengths[b])
        pos = torch.arange(max(0, min(length, width * page)))
        entry = table[b].cpu().long()[pos // page]
        res.append((starts[b], n, length - n, torch.where((entry >= 0) & (entry < pages), entry * page + pos % page, -1)))
    return res


def attention(q, k_cache, v_cache, table, lengths, starts=None, scale=None, window=0):
    """(out [T, Hq, D], bound)"""
    T, Hq, D = q.shape
    pages, page, Hkv, _ = k_cache.shape
    scale = D ** -0.5 if scale is None else scale
    h = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for first, n, before, at in places(table, lengths, starts, page, pages):
        there = torch.nonzero(at >= 0)[:, 0].to(q.device)
        if n == 0 or there.numel() == 0:
            continue
        where = at.to(q.device)[there]
        keys, values = k_cache[where // page, where % page].double(), v_cache[where // page, where % page].double()
        p = before + torch.arange(n, device=q.device)[:, None]
        seen = (there <= p) & ((there > p - window) if window else True)
        for g in range(Hq):
            k, v = keys[:, g // (Hq // Hkv)], values[:, g // (Hq // Hkv)]
            x = q[first:first + n, g].double()
            k0, bad = torch.where(k.isfinite(), k, 0.0), ~v.isfinite()
            s = x @ k.t().contiguous() * scale
            s = torch.where(seen, s, -math.inf)
            off = D * U * abs(scale) * (x.abs() @ k0.abs().t().contiguous()) + 4 * U * torch.where(seen, s, 0.0).abs()
            m = s.amax(1, keepdim=True)
            m = torch.where(m == -math.inf, 0.0, m)
            e = (s - m).exp()
            total = e.sum(1, keepdim=True)
            total = torch.where(total == 0, 1.0, total)
            w = e / total
            v0 = torch.where(bad, 0.0, v)
            o = w @ v0
            o = torch.where(seen.double() @ bad.double() > 0, math.nan, o)
            size = w @ v0.abs()
            off = (2 * off.amax(1, keepdim=True) + 4 * U * (s - m).masked_fill(~seen, 0).abs().clamp(max=200).amax(1, keepdim=True)
                   + (seen.sum(1, keepdim=True) + 64) * U)
            rounded = torch.minimum(size * h, 8 * h * (w.square() @ v0.square()).sqrt() + 2 * h * o.abs())
            if q.dtype == torch.float16:
                rounded = rounded + 2.0 ** -25 * (seen.double() @ v0.abs()) / total
            out[first:first + n, g] = o
            bound[first:first + n, g] = rounded + size * off
    return out, bound + half_step(out, q.dtype)
