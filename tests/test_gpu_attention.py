"""paged_attention against the formula in 64 bits."""
import math

import pytest
import torch

import attention_ref as A
from operators_ref import assert_close
from test_gpu_rotary import batch, log, normal

BF16, F16 = torch.bfloat16, torch.float16
pytestmark = pytest.mark.gpu


def check(device, new, lengths, page, Hq, Hkv, D, dtype, window=0, seed=0, std=2.0, padding=0, scale=None):
    from qmoe import paged_attention
    log(f"attention new={new[:8]} lengths={lengths[:8]} page={page} {Hq}/{Hkv}x{D} {dtype} window={window}")
    caches, table, lens, starts = batch(device, seed, new, lengths, page, Hkv, D, dtype)
    q = normal(device, seed + 1)(sum(new) + padding, Hq, D, std=std, dtype=dtype)
    given = starts if padding or any(n != 1 for n in new) else None
    out = paged_attention(q, *caches, table, lens, starts=given, window=window, scale=scale)
    assert out.is_contiguous()
    assert_close(out, *A.attention(q, *caches, table, lens, starts, scale, window), "attention")
    if padding:
        assert not out[sum(new):].any()
    return out


SHAPES = [(1, 1, 64), (8, 1, 128), (4, 4, 80), (15, 3, 96), (32, 2, 256), (6, 2, 192), (7, 1, 8), (64, 1, 64), (5, 5, 40),
          (24, 8, 128), (40, 2, 128)]


@pytest.mark.parametrize("Hq,Hkv,D", SHAPES)
@pytest.mark.parametrize("page", [16, 24, 64])
def test_single_tokens(device, Hq, Hkv, D, page):
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 0, 127, 128, 129, 300, 1000]
    check(device, [1] * len(lengths), lengths, page, Hq, Hkv, D, BF16, seed=D)
    check(device, [1] * len(lengths), lengths, page, Hq, Hkv, D, F16, seed=D + 1, window=50)


@pytest.mark.parametrize("lengths", [[1], [4097], [70000], [33, 50000], [2] * 200, [5000] * 17])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 1, 128), (32, 8, 64), (16, 2, 256)])
def test_single_tokens_long(device, lengths, Hq, Hkv, D):
    check(device, [1] * len(lengths), lengths, 16, Hq, Hkv, D, BF16, seed=len(lengths))


@pytest.mark.parametrize("lengths", [[99000], [131072], [60000, 1, 45000]])
@pytest.mark.parametrize("Hq,Hkv", [(8, 1), (1, 1), (6, 3)])
def test_single_tokens_many_parts(device, lengths, Hq, Hkv):
    """Heads of 64, one head's keys over nearly all workgroups."""
    check(device, [1] * len(lengths), lengths, 64, Hq, Hkv, 64, BF16)


@pytest.mark.parametrize("Hq,Hkv,D", SHAPES)
@pytest.mark.parametrize("dtype,window", [(BF16, 0), (F16, 0), (BF16, 9), (F16, 130)])
def test_several(device, Hq, Hkv, D, dtype, window):
    """A few new tokens each, none among them, more of them than are cached (rows before the start)."""
    check(device, [3, 0, 8, 1, 5, 2, 6], [3, 0, 200, 64, 1000, 66, 4], 16, Hq, Hkv, D, dtype, window, seed=D, padding=3)


@pytest.mark.parametrize("Hq,Hkv,D", SHAPES)
@pytest.mark.parametrize("dtype,window,page", [(BF16, 0, 16), (F16, 0, 24), (BF16, 70, 64), (F16, 1, 16)])
def test_chunks(device, Hq, Hkv, D, dtype, window, page):
    check(device, [97, 0, 1, 300, 64], [97, 10, 777, 500, 63], page, Hq, Hkv, D, dtype, window, seed=D, padding=5)


@pytest.mark.parametrize("new,before", [(1, 0), (2, 0), (31, 0), (32, 0), (33, 0), (63, 1), (64, 0), (65, 0), (128, 0),
                                        (129, 127), (512, 0), (1000, 3001), (2049, 0), (16, 40000), (200, 9000)])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 1, 128), (4, 4, 64), (6, 2, 256)])
def test_one_sequence(device, new, before, Hq, Hkv, D):
    for dtype, window in ((BF16, 0), (F16, 100)):
        check(device, [new], [new + before], 16, Hq, Hkv, D, dtype, window, seed=new)


@pytest.mark.parametrize("page", [1, 3, 4, 8, 100, 4096])
def test_pages(device, page):
    """Pages that end anywhere in a tile, single tokens and chunks."""
    check(device, [1] * 4, [5, 64, 333, 1201], page, 8, 2, 128, BF16, seed=page)
    check(device, [70, 3], [333, 1201], page, 8, 2, 64, F16, seed=page, window=40)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 1, 100, 6]])
@pytest.mark.parametrize("window", [0, 60])
def test_no_page(device, new, window):
    """Keys without a page are left out, in whole tiles, parts of them and to the last one."""
    from qmoe import paged_attention
    caches, table, lens, starts = batch(device, 3, new, [40, 400, 700, 64], 16, 2, 64, BF16)
    table[0, :] = -1
    table[1, :8] = -1
    table[1, 11] = caches[0].shape[0]
    table[2, ::3] = -7
    table[2, 20:40] = 1 << 30
    table[3, -1] = -1
    q = normal(device, 4)(sum(new), 8, 64, std=2.0)
    log(f"no page new={new} window={window}")
    out = paged_attention(q, *caches, table, lens, starts=starts, window=window)
    assert_close(out, *A.attention(q, *caches, table, lens, starts, None, window), "no page")
    assert not out[:new[0]].any()
    for t in (table[:, :0], torch.full_like(table, -1)):
        assert not paged_attention(q, *caches, t, lens, starts=starts, window=window).any()
    none = caches[0][:0]
    assert not paged_attention(q, none, none, table, lens, starts=starts, window=window).any()
    half = table[:, :10]  # lengths beyond the table
    out = paged_attention(q, *caches, half, lens, starts=starts, window=window)
    assert_close(out, *A.attention(q, *caches, half, lens, starts, None, window), "short table")


@pytest.mark.parametrize("new", [[1, 1, 1], [5, 1, 3], [70, 1, 33]])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 20])
def test_values_in_unseen_places(device, new, D, window):
    """NaN and infinities behind the end, before the window, on unused pages and in the keys of later
    tokens do not reach a row; a NaN that it sees does."""
    from qmoe import paged_attention
    lengths = [90, 131, 75]
    caches, table, lens, starts = batch(device, 5, new, lengths, 16, 2, D, BF16)
    used = torch.zeros(caches[0].shape[:2], dtype=torch.bool, device=device)
    sets = A.places(table, lens, starts, 16, caches[0].shape[0])
    for (first, n, before, at) in sets:
        low = max(0, before - window + 1) if window else 0
        at = at[low:].to(device)
        used[at // 16, at % 16] = True
    for c, v in zip(caches, (float("nan"), -float("inf"))):
        c[~used] = v
    caches[1][~used] = float("nan")
    first, n, before, at = sets[0]
    later = int(at[-1])  # the last token of the first sequence: its own row sees it alone
    caches[0][later // 16, later % 16, 0, 3] = float("inf")
    caches[1][later // 16, later % 16, :, 1] = float("nan")
    caches[1][later // 16, later % 16, :, D - 1] = -float("inf")
    q = normal(device, 6)(sum(new), 6, D, std=2.0)
    log(f"unseen values new={new} D={D} window={window}")
    out = paged_attention(q, *caches, table, lens, starts=starts, window=window)
    want, bound = A.attention(q, *caches, table, lens, starts, None, window)
    row = starts[1] - 1
    # (the first key head's rows score it +-inf: a weight of NaN or of 0)
    assert out[row, 3:, 1].isnan().all() and not out[row, 3:, D - 1].isfinite().any()
    keep = torch.ones(sum(new), dtype=torch.bool, device=device)
    keep[row] = False
    assert out[keep].isfinite().all()
    assert_close(out[keep], want[keep], bound[keep], "other rows")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("new", [[1], [40]])
def test_large_scores(device, dtype, new):
    """Scores far apart, rising and falling along the keys, far below zero, -inf from infinite keys; equal scores."""
    from qmoe import paged_attention
    caches, table, lens, starts = batch(device, 8, new, [1000], 16, 1, 64, dtype)
    q = normal(device, 9)(new[0], 4, 64, dtype=dtype)
    place = A.places(table, lens, starts, 16, caches[0].shape[0])[0][3].to(device)
    ramp = torch.linspace(-1, 1, 1000, device=device)
    for name, line, size in (("rising", ramp, 300.0), ("falling", -ramp, 300.0), ("low", ramp * 1e-3 - 1, 30000.0),
                             ("equal", ramp * 0, 1.0), ("steep", ramp.abs(), 6000.0)):
        log(f"large scores {name} {dtype} new={new}")
        q[..., 0], q[..., 1:] = 1.0, 0.0
        caches[0][place // 16, place % 16, 0, 0] = (line * size).to(dtype)
        out = paged_attention(q, *caches, table, lens, starts=starts, scale=1.0)
        assert_close(out, *A.attention(q, *caches, table, lens, starts, 1.0), name)
    caches[0][place[:700] // 16, place[:700] % 16, 0, 0] = -float("inf")
    out = paged_attention(q, *caches, table, lens, starts=starts, scale=1.0)
    assert_close(out, *A.attention(q, *caches, table, lens, starts, 1.0), "-inf scores")
    caches[0][place // 16, place % 16, 0, 0] = -float("inf")
    assert not paged_attention(q, *caches, table, lens, starts=starts, scale=1.0).any()


@pytest.mark.parametrize("new,lengths,Hq,Hkv,D", [([8200], [8200], 32, 8, 64), ([40, 1, 3, 17, 0, 64] * 25, [90, 500, 3, 17, 5, 129] * 25, 4, 2, 128),
                                                  ([2000, 1000, 3000, 2100], [2000, 1500, 3000, 9000], 32, 8, 64)])
def test_many_tiles(device, new, lengths, Hq, Hkv, D):
    """More tiles of rows than run at once, whole; more sequences than lanes."""
    check(device, new, lengths, 16, Hq, Hkv, D, BF16, seed=5, padding=100)


def test_layouts(device):
    """q as a slice of wider rows at any alignment, caches as views, scale 0 and below 0, tables of wider rows."""
    from qmoe import paged_attention
    caches, table, lens, starts = batch(device, 2, [3, 50], [200, 333], 16, 2, 64, BF16)
    wide = normal(device, 3)(53, 9, 75)
    for q in (wide[:, :6, :64], wide[:, 1:7, 3:67], wide[:, ::2, 5:69][:, :4], wide.transpose(1, 2)[:, :64].transpose(1, 2)[:, :8],
              wide[:1, :2, :64].expand(53, 2, 64)):
        log(f"layout {q.stride()}")
        want = A.attention(q, *caches, table, lens, starts)
        assert_close(paged_attention(q, *caches, table, lens, starts=starts), *want, "q")
    by_head = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in caches]
    both = torch.stack(caches, 1)
    spread = torch.full((2, 40), 12345, dtype=torch.int32, device=device)
    spread[:, 1:1 + table.shape[1]] = table
    for kc, vc, t in ((*by_head, table), (both[:, 0], both[:, 1], table), (caches[0], by_head[1], spread[:, 1:1 + table.shape[1]]),
                      (*caches, table.t().contiguous().t())):
        assert torch.equal(paged_attention(q, kc, vc, t, lens, starts=starts), paged_attention(q, *caches, table, lens, starts=starts))
    for scale in (0.0, -0.3):
        want = A.attention(q, *caches, table, lens, starts, scale)
        assert_close(paged_attention(q, *caches, table, lens, starts=starts, scale=scale), *want, "scale")
    none = torch.zeros((0, 4, 64), dtype=BF16, device=device)
    assert paged_attention(none, *caches, table, lens, starts=torch.zeros_like(starts)).shape == none.shape
    assert paged_attention(none, *caches, table[:0], lens[:0]).shape == none.shape


def test_far_pages(device):
    """A cache beyond 2^31 elements: its last pages, and steps that pass 32 bits."""
    from qmoe import append_kv, paged_attention
    pages = (1 << 31) // (64 * 2 * 128) + 70
    log(f"far pages: {pages}")
    k_cache, v_cache = (torch.empty((pages, 64, 2, 128), dtype=BF16, device=device) for _ in range(2))
    n = normal(device, 7)
    for new in ([1, 1], [100, 3]):
        lengths = torch.tensor([500, 130], dtype=torch.int32, device=device)
        starts = torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device=device)
        table = torch.arange(pages - 16, pages, dtype=torch.int32, device=device).view(2, 8).flip(0)
        full = torch.tensor([0, 500, 630], dtype=torch.int32, device=device)
        k, v = n(630, 2, 128), n(630, 2, 128)
        append_kv(k, v, k_cache, v_cache, table, lengths, starts=full)
        q = n(sum(new), 8, 128, std=2.0)
        out = paged_attention(q, k_cache, v_cache, table, lengths, starts=starts)
        low = table - (pages - 16)
        want = A.attention(q, k_cache[pages - 16:], v_cache[pages - 16:], low, lengths, starts)
        assert_close(out, *want, "far pages")
