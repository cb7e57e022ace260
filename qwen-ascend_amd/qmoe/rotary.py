"""Rotary positions.

Pair i of a head at position p turns by the angle p * f_i, with f_i = base^(-2i / dim). The
frequencies, worked out in double precision, are kept as 64-bit fractions of a turn, so an angle is one
integer product, which adds no error at any position; no table of cosines is kept. HIP kernel ``qmoe_rotate`` of libqmoe.so. Forward only: a
tensor that requires a gradient is refused while gradients are recorded, and one with a
forward-mode tangent.
"""
from __future__ import annotations

import math

import torch

from . import _lib

_TYPES = _lib.TYPES
D_MAX = 1024


class Rotary:
    """Frequencies and layout of rotary positions, kept by a model for all its layers.

    ``dim`` (even): how many leading elements of a head turn. ``layout``: pairs (i, i + dim/2),
    "half", or (2i, 2i + 1), "interleaved". ``scaling`` for contexts ``factor`` times as long as
    the ``original_length`` that was trained on:

    * "linear": f_i / factor;
    * "base": the base times factor^(dim / (dim - 2)), which leaves the fastest pair as it is and
      scales the slowest by the factor;
    * "parts": pairs with more than ``beta_fast`` turns within the original length stay, pairs
      with fewer than ``beta_slow`` are divided by the factor, a linear ramp over the index
      between them (YaRN); cosine and sine are multiplied by ``turn``, 0.1 ln(factor) + 1 if not given.

    ``frequencies``: dim/2 angles per position in radians, instead of all of these. ``turn``
    multiplies cosine and sine (1 but for "parts").
    """

    def __init__(self, dim, base=10000.0, *, layout="half", scaling=None, factor=1.0, original_length=None, beta_fast=32.0,
                 beta_slow=1.0, turn=None, frequencies=None, device="cuda"):
        if dim != int(dim) or not 2 <= dim <= D_MAX or dim % 2:
            raise RuntimeError(f"dim must be even, 2..{D_MAX}")
        if layout not in ("half", "interleaved"):
            raise RuntimeError("layout is 'half' or 'interleaved'")
        dim, base, factor = int(dim), float(base), float(factor)
        if frequencies is not None:
            if scaling is not None:
                raise RuntimeError("frequencies are taken as they are: no scaling")
            f = [float(v) for v in frequencies]
            if len(f) != dim // 2:
                raise RuntimeError(f"frequencies must be {dim // 2} numbers")
        else:
            f, found = self._scaled(dim, base, scaling, factor, original_length, beta_fast, beta_slow)
            turn = found if turn is None else turn
        turn = 1.0 if turn is None else float(turn)
        if not all(math.isfinite(v) for v in (*f, turn)):
            raise RuntimeError("frequencies and turn must be finite")
        self.dim, self.layout, self.turn = dim, layout, turn
        turns = [round(math.fmod(v / (2 * math.pi), 1.0) * 2.0 ** 64) % 2 ** 64 for v in f]
        self.frequencies = torch.tensor([v - (v >> 63 << 64) for v in turns], dtype=torch.int64, device=device)

    @staticmethod
    def _scaled(dim, base, scaling, factor, original_length, beta_fast, beta_slow):
        if not (math.isfinite(base) and base > 1.0):
            raise RuntimeError("base must be above 1")
        if scaling not in (None, "linear", "base", "parts"):
            raise RuntimeError("scaling is None, 'linear', 'base' or 'parts'")
        if not (math.isfinite(factor) and factor >= 1.0) or (scaling is None and factor != 1.0):
            raise RuntimeError("factor must be 1 or more, and comes with a scaling")
        if scaling == "base":
            if dim < 4:
                raise RuntimeError("scaling 'base' needs dim >= 4")
            base *= factor ** (dim / (dim - 2))
        f = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
        if scaling == "linear":
            f = [v / factor for v in f]
        if scaling != "parts":
            return f, 1.0
        if original_length is None or not original_length >= 1:
            raise RuntimeError("scaling 'parts' needs original_length")
        if not (0 < beta_slow < beta_fast and math.isfinite(beta_fast)):
            raise RuntimeError("scaling 'parts' needs 0 < beta_slow < beta_fast")
        # the (real) index whose pair makes so many turns within the original length
        low, high = (dim * math.log(original_length / (2 * math.pi * n)) / (2 * math.log(base)) for n in (beta_fast, beta_slow))
        low, high = max(math.floor(low), 0), min(math.ceil(high), dim - 1)
        for i, v in enumerate(f):
            ramp = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            f[i] = v * (1.0 - ramp) + v / factor * ramp
        return f, 0.1 * math.log(factor) + 1.0


def _heads(t, what):
    """t as rows [..., heads, D] whose elements are contiguous."""
    if t.is_neg():  # the imaginary part of a conjugate: its memory holds the other sign
        t = t.resolve_neg()
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        t = t.contiguous()
    return t


def _positions(positions, lead):
    if positions.dtype not in (torch.int32, torch.int64):
        raise RuntimeError("positions must be int32 or int64")
    if positions.shape != lead:
        raise RuntimeError(f"positions {tuple(positions.shape)} must be {tuple(lead)}, one for each token")


def _check_rotary(rotary, D):
    if not isinstance(rotary, Rotary):
        raise RuntimeError("rotary must be a Rotary")
    if rotary.dim > D:
        raise RuntimeError(f"rotary turns {rotary.dim} elements of heads of {D}")


def rotate(x, positions, rotary, *, inplace=False):
    """The heads x [..., heads, D] (bfloat16, float16 or float32) turned by their tokens' positions.

    positions [...] int32 or int64, any value; rotary: a :class:`Rotary` whose ``dim`` <= D <= 1024
    leading elements turn, the rest are copied. Returns a contiguous tensor, or with
    ``inplace=True`` x itself, written over."""
    if x.dtype not in _TYPES:
        raise RuntimeError("x must be bfloat16, float16 or float32")
    if x.dim() < 2 or not 1 <= x.shape[-1] <= D_MAX:
        raise RuntimeError(f"x must be [..., heads, D] with 1 <= D <= {D_MAX}")
    heads, D = x.shape[-2:]
    _check_rotary(rotary, D)
    _positions(positions, x.shape[:-2])
    if not _lib.operands(x, positions, rotary.frequencies):
        with torch.cuda.device(x.device):
            return rotate(x, positions, rotary, inplace=inplace)
    if inplace:
        out, rows = x, _inplace_heads(x, heads, D)
        o, o_token, o_head = rows, rows.stride(0), rows.stride(1)
        if not x.is_inference():
            torch.autograd.graph.increment_version(x)
    else:
        out = o = _lib.contiguous_like(x, x.dtype)
        rows = _heads(x, "x")
        if rows.dim() != 3:
            rows = rows.reshape(-1, heads, D) if rows.numel() else rows.new_empty((0, heads, D))
        o_token, o_head = heads * D, D
    if positions.dim() != 1 or not positions.is_contiguous():
        positions = positions.reshape(-1).contiguous()
    _lib.check(_lib.lib().qmoe_rotate(
        rows.data_ptr(), rows.stride(0), rows.stride(1), o.data_ptr(), o_token, o_head, _TYPES[x.dtype],
        positions.data_ptr(), int(positions.dtype == torch.int64), rotary.frequencies.data_ptr(), rotary.dim,
        int(rotary.layout == "interleaved"), rotary.turn, rows.shape[0], heads, D, _lib.stream_of(x)), "rotate")
    return out


def _apart(sizes, steps, width):
    """Whether runs of ``width`` elements, so many at each of these steps, lie apart."""
    for n, step in sorted(((n, s) for n, s in zip(sizes, steps) if n > 1), key=lambda v: v[1]):
        if step < width:
            return False
        width = step * (n - 1) + width
    return True


def _inplace_heads(x, heads, D):
    if x.is_neg():
        raise RuntimeError("inplace needs a tensor that is not a lazily negated view (resolve_neg())")
    try:
        rows = x if x.dim() == 3 else x.view(-1, heads, D) if x.numel() else x.new_empty((0, heads, D))
    except RuntimeError:
        raise RuntimeError("inplace needs rows of heads: leading dimensions that merge into one") from None
    if rows.numel() and ((rows.stride(2) != 1 and D != 1) or not _apart(rows.shape[:2], rows.stride()[:2], D)):
        raise RuntimeError("inplace needs heads of contiguous elements that do not overlap")
    return rows
