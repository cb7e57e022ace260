"""Norms around a block, with its gate and residual scale.

A pre-norm layer calls, around each of its blocks (:func:`qmoe.shared.moe_block` here),

    x = block_norm(h, w)                      # before the first block
    y = block(x)
    h, x = block_residual(y, h, next_weight=w)  # its residual sum and the next block's input

RMS norm in fp32, n(v; w) = v * (mean(v^2) + eps)^(-1/2) * (offset + w), each output rounded
once. HIP kernels of libqmoe.so (``qmoe_block_norm``, ``qmoe_block_residual``), one launch
per call on the current stream of the tensors' device; operands that are no rows of contiguous
elements (strided columns, dimensions that do not merge into rows, lazily negated views) are
copied first. Forward only: a tensor that requires a gradient is refused while gradients are
recorded, and one with a forward-mode tangent.
"""
from __future__ import annotations

import torch

from . import _lib

_TYPES = _lib.TYPES
H_MAX = 32768


def _rows(t, H):
    """t [..., H] as rows [n, H] whose elements are contiguous (a view where it can be one)."""
    if t.is_neg():  # the imaginary part of a conjugate: its memory holds the other sign
        t = t.resolve_neg()
    if t.dim() != 2:
        t = t.reshape(-1, H)
    if t.stride(1) != 1 and H != 1:
        t = t.contiguous()
    return t


def _check_weight(w, H, what):
    if w.dtype not in _TYPES or w.shape != (H,):
        raise RuntimeError(f"{what} must be a [{H}] tensor in bfloat16, float16 or float32")
    if w.is_neg():
        w = w.resolve_neg()
    return w if w.stride(0) == 1 or H == 1 else w.contiguous()


def _check_row_tensor(t, what):
    if t.dtype not in _TYPES:
        raise RuntimeError(f"{what} must be bfloat16, float16 or float32")
    if t.dim() < 1 or not 1 <= t.shape[-1] <= H_MAX:
        raise RuntimeError(f"{what} must be [..., H] with 1 <= H <= {H_MAX}")


def block_norm(x, weight, *, eps=1e-6, offset=0.0, out_dtype=None):
    """The norm before a block: n(x; weight) for rows x [..., H].

    ``offset`` is added to the weight (1.0 for weights stored as their distance
    from one). ``out_dtype`` is x's type, or bfloat16/float16 for a float32 x (a
    32-bit residual stream normed to the block's type). ``eps`` >= 1e-30. Returns a
    contiguous tensor of x's shape."""
    _check_row_tensor(x, "x")
    H, xt = x.shape[-1], x.dtype
    if out_dtype is None:
        out_dtype = xt
    elif out_dtype not in _TYPES or (out_dtype != xt and xt != torch.float32):
        raise RuntimeError("out_dtype must be x's type, or bfloat16 or float16 for a float32 x")
    weight = _check_weight(weight, H, "weight")
    if not _lib.operands(x, weight):
        with torch.cuda.device(x.device):
            return block_norm(x, weight, eps=eps, offset=offset, out_dtype=out_dtype)
    out = _lib.contiguous_like(x, out_dtype)
    x = _rows(x, H)
    _lib.check(_lib.lib().qmoe_block_norm(x.data_ptr(), x.stride(0), _TYPES[xt], weight.data_ptr(),
                                          _TYPES[weight.dtype], out.data_ptr(), H, _TYPES[out_dtype], x.shape[0], H, eps,
                                          offset, _lib.stream_of(x)), "block_norm")
    return out


def _gate_steps(gate, shape, H):
    """The gate as (tensor, row step, column step) of the rows of ``shape``."""
    if gate.is_neg():
        gate = gate.resolve_neg()
    if len(shape) == 2 and gate.shape == (shape[0], 1):  # one per row, the common one: no view made
        return gate, gate.stride(0), 0
    try:
        g = gate.expand(shape)
    except RuntimeError:
        raise RuntimeError(f"gate {tuple(gate.shape)} does not broadcast to {tuple(shape)}") from None
    if H == 1 or g.stride(-1) == 0:  # one per row: of a batch of sequences, a copy of a value per row at most
        g = g[..., :1].reshape(-1, 1)
        return g, g.stride(0), 0
    if g.dim() != 2:
        g = g.reshape(-1, H)
    if g.stride(1) != 1:
        g = g.contiguous()
    return g, g.stride(0), 1


def _span(t):
    """Bytes [first, past the last) that a tensor's elements lie in."""
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _other_columns(rows, t):
    """Whether t's rows lie beside those of ``rows``, as columns of the same wider rows."""
    if (t.dim() != 2 or t.dtype != rows.dtype or t.stride(1) not in (0, 1) or t.stride(0) != rows.stride(0)
            or rows.stride(0) < rows.shape[1]):
        return False
    column = (t.data_ptr() - rows.data_ptr()) // t.element_size() % rows.stride(0)
    return column >= rows.shape[1] and column + (t.shape[1] if t.stride(1) else 1) <= rows.stride(0)


def _inplace_rows(residual, H, others):
    """Rows of a residual that is written in place: a view of it, apart from each other and from
    every other operand (y may be the residual itself)."""
    if residual.is_neg():  # its memory holds the other sign
        raise RuntimeError("inplace needs a residual that is not a lazily negated view (resolve_neg())")
    rows = residual if residual.dim() == 2 else residual.view(-1, H)
    if rows.shape[0] and ((rows.stride(1) != 1 and H != 1) or (rows.stride(0) < H and rows.shape[0] > 1)):
        raise RuntimeError("inplace needs a residual of rows with contiguous elements that do not overlap")
    lo, hi = _span(rows)
    for t, itself_is_fine in others:
        if t is None:
            continue
        a, b = _span(t)
        if a < hi and lo < b and not _other_columns(rows, t):
            itself = a == lo and t.dtype == rows.dtype and t.shape == residual.shape and t.stride() == residual.stride()
            if not (itself_is_fine and itself):
                raise RuntimeError("inplace: the residual overlaps another operand")
    return rows


def block_residual(y, residual, *, post_weight=None, gate=None, gate_act=None, scale=1.0, next_weight=None,
                   eps=1e-6, offset=0.0, inplace=False):
    """What follows a block: h = residual + scale * a(gate) * p, with p = n(y; post_weight)
    (or y without one), and with ``next_weight`` the next block's input x = n(h; next_weight).

    y [..., H]; residual of y's shape and type, or float32 beside a 16-bit y. gate: any
    tensor that broadcasts to y (one value per row, per channel or per element; one per
    sequence and channel, [B, 1, H], is written out for every row first), a: its value, or its
    sigmoid for ``gate_act="sigmoid"``. The weights take ``offset`` as in
    :func:`block_norm`. Returns h (contiguous, the residual's type), or (h, x) with x in y's
    type; x is normed from h before h is rounded. ``inplace=True`` writes h over
    ``residual`` and returns that tensor."""
    _check_row_tensor(y, "y")
    H = y.shape[-1]
    if residual.shape != y.shape:
        raise RuntimeError(f"residual {tuple(residual.shape)} and y {tuple(y.shape)} do not match")
    if residual.dtype != y.dtype and residual.dtype != torch.float32:
        raise RuntimeError("residual must have y's type or float32")
    if gate_act not in (None, "sigmoid"):
        raise RuntimeError("gate_act is None or 'sigmoid'")
    if gate is not None and gate.dtype not in _TYPES:
        raise RuntimeError("gate must be bfloat16, float16 or float32")
    if gate is None and gate_act is not None:
        raise RuntimeError("gate_act needs a gate")
    if post_weight is not None:
        post_weight = _check_weight(post_weight, H, "post_weight")
    if next_weight is not None:
        next_weight = _check_weight(next_weight, H, "next_weight")
    if not _lib.operands(y, residual, post_weight, gate, next_weight):
        with torch.cuda.device(y.device):
            return block_residual(y, residual, post_weight=post_weight, gate=gate, gate_act=gate_act, scale=scale,
                                  next_weight=next_weight, eps=eps, offset=offset, inplace=inplace)
    g, g_row, g_col = (None, 0, 0) if gate is None else _gate_steps(gate, y.shape, H)
    if inplace:
        h = residual
        res = hr = _inplace_rows(residual, H, ((y, True), (gate, False), (post_weight, False), (next_weight, False)))
        ldr = ldh = res.stride(0) if res.shape[0] > 1 else H
        if not residual.is_inference():
            torch.autograd.graph.increment_version(residual)
    else:
        hr = h = _lib.contiguous_like(residual, residual.dtype)
        res = _rows(residual, H)
        ldr, ldh = res.stride(0), H
    x = None if next_weight is None else _lib.contiguous_like(y, y.dtype)
    y = _rows(y, H)
    ptr = _lib.ptr
    _lib.check(_lib.lib().qmoe_block_residual(
        y.data_ptr(), y.stride(0), _TYPES[y.dtype], res.data_ptr(), ldr,
        _TYPES[res.dtype], ptr(post_weight), 0 if post_weight is None else _TYPES[post_weight.dtype], ptr(g), g_row,
        g_col, 0 if g is None else _TYPES[g.dtype], int(gate_act == "sigmoid"), scale, hr.data_ptr(), ldh,
        ptr(next_weight), 0 if next_weight is None else _TYPES[next_weight.dtype], ptr(x), H, y.shape[0], H, eps,
        offset, _lib.stream_of(y)), "block_residual")
    return h if x is None else (h, x)
