"""paged_attention where values are infinite or NaN."""
import math

import pytest
import torch

import attention_ref as A
import test_gpu_attention as base
from test_gpu_rotary import batch, log, normal

BF16 = torch.bfloat16
INF = math.inf
pytestmark = pytest.mark.gpu

# one token, few and many; whole, in shares and in pieces that are joined
FORMS = [(1, 90), (1, 9000), (3, 700), (40, 300), (300, 9000)]


@pytest.mark.parametrize("new,before", FORMS)
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_no_weight_at_all(device, new, before, D):
    """Rows whose scores are all -inf give 0, whatever the values."""
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
