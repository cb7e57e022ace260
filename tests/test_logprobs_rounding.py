"""token_logprobs against its documented rounding bound: rows whose fp32 additions really round.

A workgroup of 4 waves takes a row in steps of 16 (fp32) or 32 (16 bits) logits per lane. The
terms of a step are summed first, then added to the lane's sum, so that a lane rounds V / 4096
times into its sum and not V / 256 times. What the bound counts, in half steps u = 2^-24 of the
sum and to first order: 31 additions within a step, one per step, 2 for exp2, 2.3 times the mean
distance to the maximum for the exponents' arguments (at most 2.3 ln V), 3 + 6 for each joining
of lanes, waves and parts; 3 more per step where the maximum rises."""
import math

import numpy as np
import pytest
import torch

U = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
# V and the distance of all logits but the first of each lane: the sums of equal terms drift with
# one rounding direction over long stretches. All distances are whole in 8 bits.
EARLY = [(1 << 22, 5.75), (1 << 22, 7.0), (1 << 22, 8.1875), (1 << 22, 9.0), (1 << 22, 10.0),
         (1 << 24, 3.25), (1 << 24, 5.75), (1 << 24, 8.1875), (1 << 24, 10.0)]


def bound(V, lp, rising):
    """The largest error of a log probability lp."""
    return ((V / 1024 if rising else V / 4096) + 128) * U + 4 * U * abs(lp)


def entropy_bound(V, entropy, rising):
    return (1 + 5 * entropy) * bound(V, 0.0, rising)


def row_of_early_maxima(V, d, dtype, device):
    """0 as the first logit of each of 256 lanes, -d in all other places."""
    x = torch.full((V,), -d, dtype=dtype, device=device)
    per = 16 // dtype.itemsize
    x[:256 * per:per] = 0
    assert x[1].item() == -d
    return x


def exact(x):
    """(ln S, entropy) of a row in 64 bits, from its largest logit."""
    l = x.double() - x.double().max()
    e = l.exp()
    s = e.sum()
    return math.log(s), (s.log() - (e * l).sum() / s).item()


def lane_sums(V, d, step):
    """One lane's fp32 sums of its V / 256 terms e^l and e^l l (base 2 inside), `step` of them summed
    first (1: one level)."""
    f = np.float32
    l = f(f(-d) * f(1.4426950408889634))
    e = np.exp2(np.float64(l)).astype(f)
    sums = []
    for first, rest in ((f(1), e), (f(0), f(e * l))):
        t = np.full(V // 256, rest, f)
        t[0] = first
        t = t.reshape(-1, step)
        inner = t[:, 0].copy()
        for i in range(1, step):
            inner = inner + t[:, i]
        sums.append(float(np.add.accumulate(inner, dtype=f)[-1]))
    return sums


@pytest.mark.parametrize("V,d", EARLY)
def test_one_level_would_be_seen(V, d):
    """The bound holds for sums in two levels and not for sums in one, on these rows."""
    want = math.log(256 * (1 + (V // 256 - 1) * math.exp(-d)))
    limit = bound(V, want, False)
    for step in (16, 32):
        assert abs(math.log(256 * lane_sums(V, d, step)[0]) - want) < limit / 2
    assert abs(math.log(256 * lane_sums(V, d, 1)[0]) - want) > limit * 1.05


def test_an_entropy_moves_by_more_than_the_sum():
    """An entropy's error is not within what the sum's additions alone allow: its bound has a factor."""
    V, d = 1 << 20, 7.9
    n = V // 256 - 1
    S, D = 256 * (1 + n * math.exp(-d)), -256 * n * d * math.exp(-d)
    want = math.log(S) - D / S
    s, w = lane_sums(V, d, 16)
    err = abs(math.log(256 * s) - math.log(2) * w / s - want)
    assert (V / 4096 + 64) * U < err <= entropy_bound(V, want, False)


def check(x, rows, rising):
    """The scores of `rows` rows that share x's memory."""
    from qmoe import token_logprobs
    V = x.numel()
    ln_s, ent = exact(x)
    ids = torch.tensor([0, V // 2, V - 1], device=x.device)
    got = token_logprobs(x.expand(rows, V), ids.expand(rows, 3))
    lp = (x[ids].double() - x.double().max() - ln_s).tolist()
    for j, want in enumerate(lp):
        err = (got.logprobs[:, j].double() - want).abs().max().item()
        assert err <= bound(V, want, rising), (j, err / U, bound(V, want, rising) / U)
    err = (got.entropy.double() - ent).abs().max().item()
    assert err <= entropy_bound(V, ent, rising), (err / U, entropy_bound(V, ent, rising) / U)
    top = token_logprobs(x.expand(rows, V), ids.expand(rows, 3), top=3)
    err = (top.top_logprobs.double() + ln_s).abs()[:, 0].max().item()
    assert err <= bound(V, -ln_s, rising)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("V,d", EARLY)
def test_early_maxima(device, V, d, dtype):
    """Whole rows on 4 waves, where a lane's sums are longest."""
    print(f"[case] early maxima V={V} d={d} {dtype}", flush=True)
    check(row_of_early_maxima(V, d, dtype, device), 513, False)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 100, 300, 513, 1100])
@pytest.mark.parametrize("V", [70001, 1 << 20, 1 << 22])
def test_rising_maxima(device, V, rows):
    """Logits that rise all along the row, so that every step moves a lane's sums to a new maximum."""
    for span in (0.5, 9.0, 40.0):
        print(f"[case] rising V={V} rows={rows} span={span}", flush=True)
        x = torch.arange(V, dtype=torch.float64, device=device).mul_(span / V).to(F32)
        check(x, rows, True)
