"""paged_attention where values are infinite or NaN: what the formula gives, wherever the keys lie; nothing from
neighbouring heads."""
import math

import pytest
import torch

import attention_ref as A
import test_gpu_attention as base
from operators_ref import assert_close
from test_gpu_rotary import batch, log, normal

BF16, F16 = torch.bfloat16, torch.float16
INF = math.inf
pytestmark = pytest.mark.gpu

# one token, few and many; whole, in shares and in pieces that are joined
FORMS = [(1, 90), (1, 9000), (3, 700), (40, 300), (300, 9000)]


def formula(q, k, v, before, window, scale):
    """sum e^(s - m) v / sum e^(s - m) over the keys that a row sees, in 64 bits: [n, Hq, D]."""
    n, Hq, D = q.shape
    p, j = before + torch.arange(n, device=q.device)[:, None], torch.arange(k.shape[0], device=q.device)
    seen = (j <= p) & ((j > p - window) if window else True)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for g in range(Hq):
        h = g // (Hq // k.shape[1])
        s = torch.where(seen, q[:, g].double() @ k[:, h].double().t().contiguous() * scale, -INF)
        m = s.amax(1, keepdim=True)
        e = torch.where(m == -INF, 0.0, (s - torch.where(m == -INF, 0.0, m)).exp())
        bad = ~v[:, h].isfinite()
        o = e @ torch.where(bad, 0, v[:, h]).double()
        for key in bad.any(1).nonzero()[:, 0].tolist():  # (0 times an infinity only where the row sees it)
            o += torch.where(seen[:, key, None], e[:, key, None] * torch.where(bad[key], v[key, h].double(), 0.0), 0.0)
        total = e.sum(1, keepdim=True)
        out[:, g] = torch.where(total == 0, 0.0, o / total)
    return out


def same_kind(out, want):
    assert torch.equal(out.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(out.isinf(), inf) and torch.equal(out[inf].double(), want[inf])


@pytest.mark.parametrize("new,before", FORMS)
@pytest.mark.parametrize("D,dtype", [(64, BF16), (64, F16), (80, BF16), (128, BF16), (192, F16), (256, BF16)])
@pytest.mark.parametrize("window", [0, 61])
def test_infinite_values(device, new, before, D, dtype, window):
    """An infinite value gives an infinity of its sign where its key has a weight, NaN where its key's score is
    -inf, and nothing where the row does not see it, in whichever tile, share or piece the key lies."""
    from qmoe import paged_attention
    log(f"infinite values {new} after {before} D={D} {dtype} window={window}")
    L = new + before
    caches, table, lens, starts = batch(device, D, [new], [L], 16, 2, D, dtype)
    q = normal(device, 1)(new, 6, D, dtype=dtype)
    q[..., 0] = 1.0
    at = A.places(table, lens, starts, 16, caches[0].shape[0])[0][3].to(device)
    spots = sorted({0, 33, before // 2, before - 70, before - 40, before - 1, before, L - 1})
    dead = [p for p in (17, before // 2 + 20, before - 60, before - 2) if p not in spots]
    values = (INF, -INF, math.nan)
    for i, p in enumerate(spots + dead):
        caches[1][at[p] // 16, at[p] % 16, i % 2, i % 8] = values[i % 3]
    for p in dead:
        caches[0][at[p] // 16, at[p] % 16, :, 0] = -INF
    keys, vals = (c[at // 16, at % 16] for c in caches)
    scale = D ** -0.5
    want = formula(q, keys, vals, before, window, scale)
    out = paged_attention(q, *caches, table, lens, starts=None if new == 1 else starts, window=window)
    same_kind(out, want)
    # the finite ones: those keys far below the others instead of at -inf
    for p in dead:
        caches[0][at[p] // 16, at[p] % 16, :, 0] = -2.0 ** 13
    fine = want.isfinite()
    ref, bound = A.attention(q, *caches, table, lens, starts, None, window)
    ref = torch.where(fine & ref.isnan(), want, ref)  # (its rule for values is coarser: a NaN for any that a row sees)
    assert_close(out[fine], ref[fine], bound[fine], "finite")


@pytest.mark.parametrize("new,before", FORMS)
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_no_weight_at_all(device, new, before, D):
    """Rows whose scores are all -inf give 0, whatever the values; with some keys' above it, a part of the keys without
    any weight brings its NaN."""
    from qmoe import paged_attention
    log(f"all scores -inf {new} after {before} D={D}")
    L = new + before
    caches, table, lens, starts = batch(device, 2, [new], [L], 16, 2, D, BF16)
    q = normal(device, 1)(new, 6, D)
    q[..., 0] = 1.0
    at = A.places(table, lens, starts, 16, caches[0].shape[0])[0][3].to(device)
    for p, v in ((0, INF), (before // 2, -INF), (before - 1, math.nan), (L - 1, INF)):
        caches[1][at[p] // 16, at[p] % 16, :, p % D] = v
    caches[0][at // 16, at % 16, 0, 0] = -INF
    given = None if new == 1 else starts
    out = paged_attention(q, *caches, table, lens, starts=given)
    assert not out[:, :3].any()
    keys, vals = (c[at // 16, at % 16] for c in caches)
    same_kind(out, formula(q, keys, vals, before, 0, D ** -0.5))
    caches[0][at[L // 2:] // 16, at[L // 2:] % 16, 0, 0] = 0.0  # and the first half still without any
    keys = caches[0][at // 16, at % 16]
    want = formula(q, keys, vals, before, 0, D ** -0.5)
    assert want[:, :3, 0].isnan().all()
    same_kind(paged_attention(q, *caches, table, lens, starts=given), want)


@pytest.mark.parametrize("new", [[1, 1, 1], [5, 1, 3], [70, 1, 33]])
@pytest.mark.parametrize("D", [8, 40, 80, 96, 136, 192])
@pytest.mark.parametrize("window", [0, 20])
def test_unseen_places_of_other_heads_sizes(device, new, D, window):
    """Heads that do not fill their rows in LDS."""
    base.test_values_in_unseen_places(device, new, D, window)


@pytest.mark.parametrize("new", [[1, 1, 1], [5, 1, 3], [70, 1, 33]])
@pytest.mark.parametrize("D", [8, 72, 80, 96, 104, 136, 192, 248])
def test_neighbouring_heads(device, new, D):
    """What the other key heads hold does not change a bit."""
    from qmoe import paged_attention
    log(f"neighbouring heads new={new} D={D}")
    caches, table, lens, starts = batch(device, 5, new, [90, 1310, 75], 16, 3, D, BF16)
    q = normal(device, 6)(sum(new), 6, D, std=2.0)
    want = paged_attention(q, *caches, table, lens, starts=starts)
    for c, v in zip(caches, (math.nan, INF)):
        c[:, :, ::2] = v
    out = paged_attention(q, *caches, table, lens, starts=starts)
    assert torch.equal(out[:, 2:4], want[:, 2:4])
    assert not out[:, :2].isfinite().any()
