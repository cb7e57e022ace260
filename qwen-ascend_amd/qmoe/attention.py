"""Attention of new tokens over a paged cache, and the cache's writer.

An attention layer calls, between its projections (q, k, v may be views of one projection's rows),

    q = append_kv(k, v, k_cache, v_cache, table, lengths, starts=starts, rotary=rotary, q=q)
    o = paged_attention(q, k_cache, v_cache, table, lengths, starts=starts)

The caches are [pages, page, Hkv, D]. A batch of B sequences is described on the device, so a
captured graph follows it: ``table`` int32 [B, width] names the page of positions [i * page, (i + 1) *
page) of a sequence (an entry outside the cache, as -1, is no page; width * page is at most 2^31 -
4096); ``lengths`` int32 [B] counts its tokens with the new ones; ``starts`` int32 [B + 1], ascending
from 0: rows [starts[b], starts[b + 1]) are its new tokens, the last ones of it. Without ``starts``
each sequence has one new token. Rows behind the last sequence are padding. HIP kernels ``qmoe_append_kv`` and ``qmoe_paged_attention`` of
libqmoe.so. Forward only: a tensor that requires a gradient is refused while gradients are
recorded, and one with a forward-mode tangent.
"""
from __future__ import annotations

import torch

from . import _lib
from .rotary import _apart, _check_rotary, _heads, _positions

_TYPES = _lib.TYPES
_bump = torch.autograd.graph.increment_version


def _check_batch(table, lengths, starts, T):
    if table.dtype != torch.int32 or table.dim() != 2:
        raise RuntimeError("table must be int32 [B, width]")
    B = table.shape[0]
    if lengths.dtype != torch.int32 or lengths.shape != (B,):
        raise RuntimeError(f"lengths must be int32 [{B}]")
    if starts is None:
        if T != B:
            raise RuntimeError(f"{T} new tokens for {B} sequences need starts")
    elif starts.dtype != torch.int32 or starts.shape != (B + 1,):
        raise RuntimeError(f"starts must be int32 [{B + 1}]")


def _cache_steps(k_cache, v_cache, dtype, Hkv, D):
    """Element steps (page, place, head) of both caches, checked; whether both are contiguous."""
    if k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise RuntimeError("the caches must have the new tokens' type")
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise RuntimeError("the caches must be [pages, page, Hkv, D], both alike")
    if shape[2] != Hkv or shape[3] != D or shape[1] < 1:
        raise RuntimeError(f"caches {tuple(shape)} do not match heads [{Hkv}, {D}]")
    if k_cache.is_neg() or v_cache.is_neg():
        raise RuntimeError("the elements of a cached head must be contiguous, and no lazily negated view")
    if k_cache.is_contiguous() and v_cache.is_contiguous():
        steps = (shape[1] * Hkv * D, Hkv * D, D)
        return steps, steps, True
    for c in (k_cache, v_cache):
        if c.stride(3) != 1 and D != 1:
            raise RuntimeError("the elements of a cached head must be contiguous, and no lazily negated view")
    return _steps(k_cache), _steps(v_cache), False


def _steps(c):
    """Element steps of a cache's pages, places and heads (0 where there is one)."""
    return [s if n > 1 else 0 for n, s in zip(c.shape[:3], c.stride())]


def _rows(t):
    """An int32 tensor whose last dimension is contiguous."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def append_kv(k, v, k_cache, v_cache, table, lengths, *, starts=None, rotary=None, positions=None, q=None):
    """Writes the new tokens' keys (turned by ``rotary``, if given) and values to their places in
    the caches, in place; a token without a page, or behind the last sequence, is left out.

    k, v [T, Hkv, D] in the caches' type (bfloat16, float16 or float32), D <= 1024. ``positions`` int32 or
    int64 [T]: the positions that the heads turn by, if not those in the sequences (which they are
    stored at in any case). q [T, Hq, D]: queries, turned alike in the same launch;
    returns them as a new contiguous tensor, None without q. Queries behind the last sequence turn as
    at position 0. No two tokens may have one place, and k, v and q must not overlap the caches."""
    if k.dtype not in _TYPES or k.dim() != 3 or not 1 <= k.shape[2] <= 1024:
        raise RuntimeError("k must be [T, Hkv, D] in bfloat16, float16 or float32 with 1 <= D <= 1024")
    T, Hkv, D = k.shape
    if v.dtype != k.dtype or v.shape != k.shape or Hkv < 1:
        raise RuntimeError("v must have k's type and shape, and heads")
    k_steps, v_steps, contiguous = _cache_steps(k_cache, v_cache, k.dtype, Hkv, D)
    if not contiguous:
        for c in (k_cache, v_cache):
            if c.numel() and not _apart(c.shape[:3], c.stride()[:3], D):
                raise RuntimeError("the places of a cache must not overlap")
    _check_batch(table, lengths, starts, T)
    if q is not None and (q.dtype != k.dtype or q.dim() != 3 or q.shape[0] != T or q.shape[2] != D):
        raise RuntimeError(f"q must be [{T}, Hq, {D}] in k's type")
    if rotary is not None:
        _check_rotary(rotary, D)
    if positions is not None:
        if rotary is None:
            raise RuntimeError("positions need a rotary")
        _positions(positions, (T,))
    frequencies = None if rotary is None else rotary.frequencies
    if not _lib.operands(k, v, k_cache, v_cache, table, lengths, starts, positions, q, frequencies):
        with torch.cuda.device(k.device):
            return append_kv(k, v, k_cache, v_cache, table, lengths, starts=starts, rotary=rotary, positions=positions, q=q)
    for c in (k_cache, v_cache):
        if not c.is_inference():
            _bump(c)
    k, v = _heads(k, "k"), _heads(v, "v")
    (k_token, k_head, _), (v_token, v_head, _) = k.stride(), v.stride()
    lengths, table = lengths.contiguous(), _rows(table)
    starts = None if starts is None else starts.contiguous()
    positions = None if positions is None else positions.contiguous()
    out, Hq, q_token, q_head = None, 0, 0, 0
    if q is not None:
        out, q, Hq = q.new_empty(q.shape), _heads(q, "q"), q.shape[1]
        q_token, q_head, _ = q.stride()
    ptr = _lib.ptr
    some = q if Hq else None  # heads or none
    dim, interleaved, turn = (0, 0, 1.0) if rotary is None else (rotary.dim, int(rotary.layout == "interleaved"), rotary.turn)
    _lib.check(_lib.lib().qmoe_append_kv(
        k.data_ptr(), k_token, k_head, v.data_ptr(), v_token, v_head, ptr(some), q_token, q_head,
        None if some is None else out.data_ptr(), _TYPES[k.dtype], k_cache.data_ptr(), *k_steps,
        v_cache.data_ptr(), *v_steps, table.data_ptr(), table.stride(0), table.shape[1], lengths.data_ptr(),
        ptr(starts), ptr(positions), int(positions is not None and positions.dtype == torch.int64), ptr(frequencies), dim,
        interleaved, turn, T, table.shape[0], Hq, Hkv, D, k_cache.shape[1], k_cache.shape[0], _lib.stream_of(k)), "append_kv")
    return out


def paged_attention(q, k_cache, v_cache, table, lengths, *, starts=None, scale=None, window=0):
    """Causal attention of the new tokens q [T, Hq, D] over the caches; returns [T, Hq, D].

    The caches hold the new tokens' keys and values too (:func:`append_kv`). The row of a token at
    position p sees the keys up to p, with a ``window`` > 0 only the last ``window`` of them, and
    none without a page. bfloat16 or float16; D <= 256 a multiple of 8; query heads [h G, (h + 1) G) share
    key head h, G = Hq / Hkv <= 64. A page of a cache spans fewer than 2^30 elements; with ``starts``,
    T Hq / 128 + (B + 1) Hkv < 2^24 - 768. ``scale``: D^-0.5 if not given. Scores, softmax and the output's sums are
    fp32; the weights e^(s - m) are rounded to q's type for their product with the values, each
    output once. A row that sees no key, or whose scores are all -inf, gives 0, and so do rows behind
    the last sequence; else an infinite value that it sees gives an infinity, or, as 0 times it, NaN where the key's
    score is -inf or its weight too small for the type. What lies at a place that a row does not see, NaN
    too, does not reach it."""
    if q.dtype not in (torch.bfloat16, torch.float16) or q.dim() != 3:
        raise RuntimeError("q must be [T, Hq, D] in bfloat16 or float16")
    T, Hq, D = q.shape
    if not 8 <= D <= 256 or D % 8:
        raise RuntimeError("D must be a multiple of 8, 8..256")
    if k_cache.dim() != 4:
        raise RuntimeError("the caches must be [pages, page, Hkv, D], both alike")
    Hkv = k_cache.shape[2]
    if Hkv < 1 or Hq < 1 or Hq % Hkv or Hq // Hkv > 64 or Hq > 4096:
        raise RuntimeError(f"{Hq} query heads cannot share {Hkv} key heads, at most 64 each and 4096 in all")
    if T * Hq >= 1 << 31:
        raise RuntimeError("q must have fewer than 2^31 rows of heads")
    k_steps, v_steps, contiguous = _cache_steps(k_cache, v_cache, q.dtype, Hkv, D)
    k_ptr, v_ptr = k_cache.data_ptr(), v_cache.data_ptr()
    if (k_ptr | v_ptr) & 15 or not (contiguous or all(s % 8 == 0 for s in (*k_steps, *v_steps))):
        raise RuntimeError("cached heads must be 16-byte aligned")
    _check_batch(table, lengths, starts, T)
    if window != int(window) or not 0 <= window <= 1 << 30:
        raise RuntimeError("window must be 0 (none) or a number of tokens up to 2^30")
    if not _lib.operands(q, k_cache, v_cache, table, lengths, starts):
        with torch.cuda.device(q.device):
            return paged_attention(q, k_cache, v_cache, table, lengths, starts=starts, scale=scale, window=window)
    out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape)
    q, table, lengths = _heads(q, "q"), _rows(table), lengths.contiguous()
    q_token, q_head, _ = q.stride()
    starts = None if starts is None else starts.contiguous()
    L, B, page, width = _lib.lib(), table.shape[0], k_cache.shape[1], table.shape[1]
    nbytes = L.qmoe_paged_attention_workspace(T, B, Hq, Hkv, D, page, width, int(starts is None))
    # from the caching allocator: aligned, its own in every graph
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    ptr = _lib.ptr
    _lib.check(L.qmoe_paged_attention(
        q.data_ptr(), q_token, q_head, k_ptr, *k_steps, v_ptr, *v_steps, _TYPES[q.dtype], table.data_ptr(),
        table.stride(0), width, lengths.data_ptr(), ptr(starts),
        out.data_ptr(), T, B, Hq, Hkv, D, page, k_cache.shape[0], D ** -0.5 if scale is None else float(scale), int(window),
        ptr(ws), nbytes, _lib.stream_of(q)), "paged_attention")
    return out
