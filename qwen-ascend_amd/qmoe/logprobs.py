"""Log probabilities of given tokens, with entropy and top alternatives.

What follows the lm_head projection (a :class:`qmoe.DenseW8`, ``fnx/load.py:189-201``):
the score of the tokens of a prompt, or of the ones sampled, beside the most likely ones.
One pass over the logits with the running maximum and sums of the softmax, on the HIP kernels
of libqmoe.so (``qmoe_token_logprobs``); nothing of the logits' size is written. Forward only:
a tensor that requires a gradient is refused while gradients are recorded, and one with a
forward-mode tangent.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib

_TYPES = _lib.TYPES
TOP_MAX = 32


class TokenLogprobs(NamedTuple):
    logprobs: Optional[torch.Tensor]      # fp32, the tokens' shape; None without tokens
    entropy: torch.Tensor                 # fp32 [...]
    top_ids: Optional[torch.Tensor]       # int64 [..., top]; None for top = 0
    top_logprobs: Optional[torch.Tensor]  # fp32 [..., top]; None for top = 0


def token_logprobs(logits, tokens=None, *, top=0, allowed=None):
    """Scores of the softmax over rows of logits [..., V] (bfloat16, float16 or float32).

    tokens int64 [...] or [..., m] (m <= 2^30 given tokens for each row): their log
    probabilities; a negative token scores 0 (padding), one that is not allowed -inf, one
    from V on NaN. The entropy of each row. The ``top`` <= 32 most likely tokens in order
    (equal logits: the lower id first) with their log probabilities; where fewer than ``top``
    have a logit above -inf, id -1 and -inf fill up.

    allowed: bool [V] or of the logits' shape; where it is False a token is out, whatever its
    logit holds. A row with no token left: its tokens -inf, entropy 0. A row with NaN or +inf
    at an allowed place has no distribution: NaN (padding still 0) and ids -1. The sums are fp32,
    in two levels. With B = V / 1024 + 128 half steps (2^-24 each), to first order: a row's sum is
    off by at most B of it, a log probability by at most B and four half steps of its own size, an
    entropy E by at most (1 + 5 E) B; by far less as a rule. (V / 1024 is the cost of a maximum that
    rises all along the row, at most four roundings a step of at least 4096 logits; where it comes
    early it is V / 4096.)
    """
    if logits.dtype not in _TYPES:
        raise RuntimeError("logits must be bfloat16, float16 or float32")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= 1 << 30:
        raise RuntimeError("logits must be [..., V] with 1 <= V <= 2^30")
    lead, V = logits.shape[:-1], logits.shape[-1]
    top = int(top)
    if not 0 <= top <= TOP_MAX:
        raise RuntimeError(f"top must be 0..{TOP_MAX}")
    m = 0
    if tokens is not None:
        if tokens.dtype != torch.int64:
            raise RuntimeError("tokens must be int64")
        if tokens.shape == lead:
            m = 1
        elif tokens.dim() == len(lead) + 1 and tokens.shape[:-1] == lead:
            m = tokens.shape[-1]
        else:
            raise RuntimeError(f"tokens {tuple(tokens.shape)} do not match logits {tuple(logits.shape)}")
        if m > 1 << 30:
            raise RuntimeError("tokens must be at most 2^30 for each row")
    if allowed is not None and (allowed.dtype != torch.bool or allowed.shape not in ((V,), logits.shape)):
        raise RuntimeError("allowed must be bool [V] or of the logits' shape")
    if not _lib.operands(logits, tokens, allowed):
        with torch.cuda.device(logits.device):
            return token_logprobs(logits, tokens, top=top, allowed=allowed)
    x = logits if logits.dim() == 2 else logits.reshape(-1, V)
    if x.is_neg():  # the imaginary part of a conjugate: its memory holds the other sign
        x = x.resolve_neg()
    if x.stride(1) != 1 and V != 1:
        x = x.contiguous()
    T = x.shape[0]
    if T >= 1 << 31:
        raise RuntimeError("logits must have fewer than 2^31 rows")
    lda = 0
    if allowed is not None:
        if allowed.dim() > 1:
            allowed = allowed if allowed.dim() == 2 else allowed.reshape(-1, V)
            lda = allowed.stride(0)
        if allowed.stride(-1) != 1 and V != 1:
            allowed = allowed.contiguous()
            lda = V if allowed.dim() > 1 else 0
    logprobs = top_ids = top_lp = ws = None
    if tokens is not None:
        tokens = tokens.contiguous()
        logprobs = torch.empty_like(tokens, dtype=torch.float32)
    entropy = x.new_empty(lead, dtype=torch.float32)
    if top:
        top_ids = x.new_empty((*lead, top), dtype=torch.int64)
        top_lp = torch.empty_like(top_ids, dtype=torch.float32)
    L = _lib.lib()
    kind, ptr = _TYPES[x.dtype], _lib.ptr
    nbytes = L.qmoe_token_logprobs_workspace(T, V, kind, top)
    if nbytes:
        ws = x.new_empty(nbytes, dtype=torch.uint8)  # from the caching allocator: aligned, its own in every graph
    _lib.check(L.qmoe_token_logprobs(x.data_ptr(), x.stride(0), kind, ptr(tokens), m, ptr(allowed), lda, T, V,
                                     ptr(logprobs), entropy.data_ptr(), top, ptr(top_ids), ptr(top_lp), ptr(ws), nbytes,
                                     _lib.stream_of(x)), "token_logprobs")
    return TokenLogprobs(logprobs, entropy, top_ids, top_lp)
