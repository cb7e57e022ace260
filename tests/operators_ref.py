"""The norms around a block and the token log probabilities in 64 bits, each with the largest
error that fp32 arithmetic and the output's rounding allow.

u = 2^-24 is fp32's half step. A norm: the squares and their sum in chains of at most H/64
(positive terms), half of that through the root, and a dozen operations; then half a step of
the output's type. Log probabilities: sums in chains of at most V/256 terms, exponents whose
argument is off by two half steps, a logarithm."""
import torch

U = 2.0 ** -24


def half_step(exact, dtype):
    f = torch.finfo(dtype)
    return exact.abs() * (f.eps / 2) * (1 + 2.0 ** -8) + f.smallest_normal * f.eps


def norm(v, w, eps, offset):
    """(n(v; w), its fp32 error bound)"""
    out = v * (v.square().mean(-1, keepdim=True) + eps).rsqrt() * (w.double() + offset)
    return out, out.abs() * (v.shape[-1] / 128 + 16) * U


def block_norm(x, w, eps=1e-6, offset=0.0, out_dtype=None):
    out, err = norm(x.double(), w, eps, offset)
    return out, err + half_step(out, out_dtype or x.dtype)


def block_residual(y, residual, post_weight=None, gate=None, gate_act=None, scale=1.0, next_weight=None, eps=1e-6,
                   offset=0.0):
    """[(h, bound)] or [(h, bound), (x, bound)]"""
    p = y.double()
    err = torch.zeros_like(p)
    if post_weight is not None:
        p, err = norm(p, post_weight, eps, offset)
    if gate is not None:
        g = gate.double().expand(p.shape)
        if gate_act == "sigmoid":
            # relative (|g| + 8) half steps; past |g| = 104 fp32 holds exactly 0 or 1, and a value
            # below fp32's normal range may be taken as 0
            err = err + p.abs() * (g.abs().clamp(max=104) + 8) * U + p.abs() * 2.0 ** -126
            g = g.sigmoid()
        p, err = p * g, err * g.abs()
    p, err = scale * p, err * abs(scale)
    r = residual.double()
    h = r + p
    err = err + 4 * U * (r.abs() + p.abs())
    res = [(h, err + half_step(h, residual.dtype))]
    if next_weight is not None:
        x, rel = norm(h, next_weight, eps, offset)
        inv = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
        w = (next_weight.double() + offset).abs()
        moved = err * inv
        res.append((x, moved * w + x.abs() * moved.amax(-1, keepdim=True) + rel + half_step(x, y.dtype)))
    return res


def token_logprobs(logits, tokens=None, top=0, allowed=None):
    """((logprobs, bound), (entropy, bound), ids, (top_logprobs, bound)) by the documented rules."""
    V = logits.shape[-1]
    x = logits.reshape(-1, V).double()
    T = x.shape[0]
    if allowed is not None:
        x = torch.where(allowed.expand(logits.shape).reshape(-1, V), x, -float("inf"))
    broken = (x.isnan() | (x == float("inf"))).any(1, keepdim=True)
    empty = (x == -float("inf")).all(1, keepdim=True)
    fine = torch.where(broken | empty, 0.0, x)
    m = fine.amax(1, keepdim=True)
    d = fine - m
    s = d.exp().sum(1, keepdim=True)
    logs = s.log()
    nan = torch.full_like(s, float("nan"))
    base = (V / 256 + 64) * U
    p = d.exp() / s
    ent = -(p * torch.where(p > 0, p.log(), 0.0)).sum(1, keepdim=True)
    ent_err = base * (1 + ent + logs)
    ent = torch.where(broken, nan, torch.where(empty, 0.0, ent))

    def score(ids):  # ids in range
        lp = torch.where(empty, -float("inf"), x.gather(1, ids)) - torch.where(empty, 0.0, m) - torch.where(empty, 0.0, logs)
        err = base + U * 2 * (d.gather(1, ids).abs().nan_to_num_(posinf=0.0) + logs)
        return torch.where(broken, nan, lp), err

    res = [None, (ent.reshape(logits.shape[:-1]), ent_err.reshape(logits.shape[:-1])), None, None]
    if tokens is not None:
        t = tokens.reshape(T, -1)
        lp, err = score(t.clamp(0, V - 1))
        lp = torch.where(t >= V, nan, lp)
        lp = torch.where(t < 0, 0.0, lp)
        res[0] = (lp.reshape(tokens.shape), err.reshape(tokens.shape))
    if top:
        k = min(top, V)
        key = torch.where(x.isnan(), 0.0, x)
        ids = torch.sort(key, dim=1, descending=True, stable=True)[1][:, :k]
        lp, err = score(ids)
        ids = torch.where(broken | (x.gather(1, ids) == -float("inf")), -1, ids)
        if k < top:
            pad = (T, top - k)
            ids = torch.cat([ids, torch.full(pad, -1, device=ids.device)], 1)
            lp = torch.cat([lp, torch.where(broken, nan, -float("inf")).expand(pad)], 1)
            err = torch.cat([err, torch.zeros(pad, device=err.device, dtype=err.dtype)], 1)
        shape = (*logits.shape[:-1], top)
        res[2], res[3] = ids.reshape(shape), (lp.reshape(shape), err.reshape(shape))
    return res


def assert_close(got, exact, bound, what):
    """Within the bound where the value is finite; the same NaN and infinities elsewhere. A
    value past the type's largest may round to infinity."""
    assert got.shape == exact.shape, (what, got.shape, exact.shape)
    g, e = got.double(), exact
    big = torch.finfo(got.dtype).max
    assert torch.equal(g.isnan(), e.isnan()), f"{what}: NaN at other places"
    over = e.abs() > big * (1 - torch.finfo(got.dtype).eps)
    same = e.isnan() | (g == e) | (over & (g.sign() == e.sign()) & (g.abs() >= big * (1 - torch.finfo(got.dtype).eps)))
    bad = ~same & ~(e.isfinite() & ((g - e).abs() <= bound))
    if bad.any():
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {at}: "
                             f"{g[at].item()!r} for {e[at].item()!r}, bound {bound[at].item()!r}")
