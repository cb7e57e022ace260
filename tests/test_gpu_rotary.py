"""rotate and append_kv against the formulas in 64 bits."""
import pytest
import torch

import attention_ref as A
from operators_ref import assert_close

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
pytestmark = pytest.mark.gpu


def log(msg):
    print(f"[case] {msg}", flush=True)


def normal(device, seed):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return lambda *shape, std=1.0, dtype=BF16: (torch.randn(shape, generator=g, device=device) * std).to(dtype)


@pytest.mark.parametrize("T,heads,D,rd", [(1, 1, 2, 2), (1, 32, 128, 128), (3, 5, 64, 32), (7, 1, 80, 80), (2, 3, 90, 54),
                                          (65, 7, 33, 10), (4, 2, 256, 64), (1030, 16, 128, 128), (2, 64, 96, 96),
                                          (1, 3, 1024, 1024), (2, 2, 1023, 1022), (5, 9, 16, 2), (9, 4, 1024, 2),
                                          (2, 2, 513, 512), (3000, 3, 192, 96)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotate(device, T, heads, D, rd, dtype, layout):
    from qmoe import Rotary, rotate
    log(f"rotate T={T} heads={heads} D={D} rd={rd} {dtype} {layout}")
    x = normal(device, T + D)(T, heads, D, dtype=dtype)
    positions = torch.randint(-(1 << 24), 1 << 24, (T,), device=device, generator=torch.Generator(device=device).manual_seed(T))
    positions[0] = 0 if T > 1 else positions[0]
    r = Rotary(rd, 5.0e5, layout=layout, device=device)
    f, turn = A.frequencies(rd, 5.0e5)
    keep = x.clone()
    out = rotate(x, positions, r)
    assert out.is_contiguous() and torch.equal(x, keep)
    assert_close(out, *A.rotate(x, positions, f, turn, layout), "rotate")
    assert torch.equal(out[..., rd:], x[..., rd:])
    assert torch.equal(rotate(x, positions.int(), r), out)
    version = x._version
    again = rotate(x, positions, r, inplace=True)
    assert again is x and x._version > version and torch.equal(x, out)


@pytest.mark.parametrize("scaling,kw", [("linear", dict(factor=8.0)), ("base", dict(factor=4.0)),
                                        ("parts", dict(factor=16.0, original_length=4096)),
                                        ("parts", dict(factor=2.0, original_length=100, beta_fast=8.0, beta_slow=0.5)),
                                        ("parts", dict(factor=40.0, original_length=4096, turn=1.0))])
@pytest.mark.parametrize("rd", [4, 64, 128])
def test_scalings(device, scaling, kw, rd):
    from qmoe import Rotary, rotate
    log(f"scaling {scaling} {kw} rd={rd}")
    x = normal(device, rd)(300, 2, 128, dtype=F32)
    positions = torch.arange(300, device=device) * 997
    for base in (1.0e4, 1.0e6):
        f, turn = A.frequencies(rd, base, scaling, kw["factor"], kw.get("original_length"), kw.get("beta_fast", 32.0),
                                kw.get("beta_slow", 1.0))
        turn = kw.get("turn", turn)
        r = Rotary(rd, base, scaling=scaling, device=device, **kw)
        assert r.turn == pytest.approx(turn)
        assert_close(rotate(x, positions, r), *A.rotate(x, positions, f, turn, "half"), scaling)
        same = Rotary(rd, frequencies=f.tolist(), turn=turn, device=device)
        assert (same.frequencies - r.frequencies).abs().max() <= 2 ** 14
    back = Rotary(rd, frequencies=(-f).tolist(), turn=1 / turn, device=device)  # the inverse
    assert_close(rotate(rotate(x, positions, r), positions, back), x.double(), 64 * A.U * (x.abs() + 4.0).double(), "back")


def test_rotate_layouts(device):
    """Heads cut out of wider rows at any alignment, leading dimensions, shared rows, strided elements; in place
    where they lie apart."""
    from qmoe import Rotary, rotate
    n = normal(device, 3)
    r = Rotary(32, device=device)
    f, turn = A.frequencies(32, 1.0e4)
    wide = n(6, 10, 100)
    views = [wide[:, :, :64], wide[:, 3:5, 5:70], wide[::2, :, 1:97], wide.view(2, 3, 10, 100), wide.transpose(0, 1),
             wide[:, :, ::2], wide[:1].expand(4, 10, 100), wide[:, :1].expand(6, 4, 100), wide[0],
             wide.view(3, 2, 10, 100).transpose(0, 1)]
    for i, x in enumerate(views):
        log(f"layout {i} {tuple(x.shape)} {x.stride()}")
        positions = torch.randint(0, 5000, x.shape[:-2], device=device)
        before = wide.clone()
        want, bound = A.rotate(x, positions, f, turn, "half")
        assert_close(rotate(x, positions, r), want, bound, f"layout {i}")
        assert torch.equal(wide, before)
        if i in (0, 1, 2, 3, 4, 8):
            assert rotate(x, positions, r, inplace=True) is x
            assert_close(x, want, bound, f"layout {i} in place")
            wide.copy_(before)
        else:
            with pytest.raises(RuntimeError, match="inplace"):
                rotate(x, positions, r, inplace=True)
    for shape in ((0, 4, 64), (3, 0, 64), (2, 0, 4, 64)):
        x = torch.empty(shape, device=device)
        p = torch.zeros(shape[:-2], dtype=torch.int64, device=device)
        assert rotate(x, p, r).shape == shape and rotate(x, p, r, inplace=True) is x
    spread = torch.arange(0, 4000, 500, device=device)
    x = n(4, 2, 64)
    assert torch.equal(rotate(x, spread[::2], r), rotate(x, spread[::2].contiguous(), r))


def test_rotate_values(device):
    """Infinities, NaN and the largest values stay in their own pairs."""
    from qmoe import Rotary, rotate
    r = Rotary(16, device=device)
    for dtype in (BF16, F16, F32):
        x = normal(device, 9)(3, 2, 24, dtype=dtype)
        x[0, 0, 1], x[1, 1, 9], x[2, 0, 20] = float("nan"), float("inf"), float("nan")
        out = rotate(x, torch.tensor([5, 7, 11], device=device), r)
        bad = ~out.isfinite()
        want = torch.zeros_like(bad)
        want[0, 0, [1, 9]] = want[1, 1, [1, 9]] = want[2, 0, 20] = True
        assert torch.equal(bad, want)
        zero = rotate(x, torch.zeros(3, dtype=torch.int32, device=device), r)
        fine = ~want
        assert torch.equal(zero[fine], x[fine])


def batch(device, seed, new, lengths, page, Hkv, D, dtype, spare=3, width=None):
    """Caches of random pages and values, with the sequences' tables."""
    g = torch.Generator(device=device).manual_seed(seed)
    pages = [-(-max(n, 0) // page) for n in lengths]
    count = sum(pages) + spare
    order = torch.randperm(count, generator=g, device=device).int()
    table = torch.full((len(new), width or max(1, *pages)), -1, dtype=torch.int32, device=device)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    caches = [torch.randn((count, page, Hkv, D), generator=g, device=device).to(dtype) for _ in range(2)]
    starts = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=device)
    return caches, table, torch.tensor(lengths, dtype=torch.int32, device=device), starts


def appended(k, v, q, caches, table, lengths, starts, f, turn, layout, positions=None, rotary=True):
    """[(k_cache, bound), (v_cache, 0), (q, bound)]"""
    pages, page = caches[0].shape[:2]
    want = [c.double() for c in caches]
    err = torch.zeros_like(want[0])
    T = k.shape[0]
    pos = torch.zeros(T, dtype=torch.int64, device=k.device)
    sets = A.places(table, lengths, starts, page, pages)
    for first, n, before, _ in sets:
        pos[first:first + n] = before + torch.arange(n, device=k.device)
    by = pos if positions is None else positions
    turned = lambda x: A.rotate(x, by, f, turn, layout) if rotary else (x.double(), torch.zeros_like(x).double())
    kt, ke = turned(k)
    for first, n, before, at in sets:
        for i in range(n):
            p = before + i
            if 0 <= p < at.shape[0] and at[p] >= 0:
                place = (int(at[p]) // page, int(at[p]) % page)
                want[0][place], err[place], want[1][place] = kt[first + i], ke[first + i], v[first + i].double()
    return (want[0], err), (want[1], torch.zeros_like(err)), (None if q is None else turned(q))


CASES = [  # new, lengths, page, Hq, Hkv, D, rd
    ([1], [1], 16, 1, 1, 64, 64), ([1] * 5, [1, 17, 16, 64, 300], 16, 8, 2, 128, 128), ([3, 0, 1, 40], [3, 5, 33, 80], 16, 6, 3, 80, 80),
    ([100], [357], 24, 4, 4, 96, 48), ([1] * 70, list(range(1, 71)), 1, 2, 1, 32, 32), ([7, 9], [7, 1000], 128, 5, 1, 256, 64),
    ([5, 2], [3, 1], 8, 2, 2, 40, 10), ([130] * 2, [130, 131], 32, 1, 1, 33, 6), ([1] * 3, [0, -4, 9], 4, 2, 2, 64, 64),
]


@pytest.mark.parametrize("new,lengths,page,Hq,Hkv,D,rd", CASES)
@pytest.mark.parametrize("dtype,layout", [(BF16, "half"), (F16, "interleaved"), (F32, "half")])
def test_append(device, new, lengths, page, Hq, Hkv, D, rd, dtype, layout):
    from qmoe import Rotary, append_kv
    log(f"append new={new[:8]} lengths={lengths[:8]} page={page} {Hq}/{Hkv}x{D} rd={rd} {dtype} {layout}")
    caches, table, lens, starts = batch(device, sum(new), new, lengths, page, Hkv, D, dtype)
    T = sum(new) + (2 if any(n != 1 for n in new) else 0)  # two rows of padding behind the last sequence
    n = normal(device, T)
    qkv = n(T, Hq + 2 * Hkv, D, dtype=dtype)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    given = None if T == len(new) and all(m == 1 for m in new) else starts
    r = Rotary(rd, layout=layout, device=device)
    f, turn = A.frequencies(rd, 1.0e4)
    want = appended(k, v, q, caches, table, lens, starts, f, turn, layout)
    got = [c.clone() for c in caches]
    version = got[0]._version
    out = append_kv(k, v, *got, table, lens, starts=given, rotary=r, q=q)
    assert out.is_contiguous() and got[0]._version > version
    for a, w, name in zip((*got, out), want, ("k_cache", "v_cache", "q")):
        assert_close(a, *w, name)
    # positions of their own; without q; without a rotary
    positions = torch.arange(T, device=device) * 31 - 100
    want = appended(k, v, q, caches, table, lens, starts, f, turn, layout, positions)
    got = [c.clone() for c in caches]
    out = append_kv(k, v, *got, table, lens, starts=given, rotary=r, positions=positions.int(), q=q)
    for a, w, name in zip((*got, out), want, ("k_cache", "v_cache", "q")):
        assert_close(a, *w, name)
    got = [c.clone() for c in caches]
    assert append_kv(k, v, *got, table, lens, starts=given) is None
    want = appended(k, v, None, caches, table, lens, starts, f, turn, layout, rotary=False)
    for a, w in zip(got, want):
        assert_close(a, *w, "copied")


def test_append_pages(device):
    """Entries that name no page leave their tokens out, also at the ends of the range; caches as views (heads
    before places, keys and values in one tensor)."""
    from qmoe import append_kv
    n = normal(device, 1)
    k, v = n(40, 2, 16), n(40, 2, 16)
    starts = torch.tensor([0, 25, 40], dtype=torch.int32, device=device)
    lengths = torch.tensor([25, 30], dtype=torch.int32, device=device)
    table = torch.tensor([[2, -1, 5, 9], [6, 1 << 30, -(1 << 31), 0]], dtype=torch.int32, device=device)
    both = torch.zeros((6, 2, 2, 8, 16), dtype=BF16, device=device)  # page, keys or values, head, place
    caches = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    log("append: pages out of range")
    append_kv(k, v, *caches, table, lengths, starts=starts)
    want = torch.zeros_like(both)
    for c, x in enumerate((k, v)):
        want[2, c] = x[0:8].transpose(0, 1)
        want[5, c] = x[16:24].transpose(0, 1)
        want[0, c, :, :6] = x[34:40].transpose(0, 1)  # positions 24..29 of the second sequence
    assert torch.equal(both, want)
    none = torch.zeros((0, 8, 2, 16), dtype=BF16, device=device)
    append_kv(k, v, none, none.clone(), table, lengths, starts=starts)
    append_kv(k, v, *caches, table[:, :0], lengths, starts=starts)
    assert torch.equal(both, want)
    empty = k[:0]
    append_kv(empty, empty, *caches, table, lengths, starts=torch.zeros_like(starts))
    append_kv(empty, empty, *caches, table[:0], lengths[:0], starts=starts[:1])
    assert torch.equal(both, want)
