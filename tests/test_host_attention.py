"""What the rotary and paged-cache operators refuse, and their references (CPU only)."""
import math

import pytest
import torch

import attention_ref as A
import operators_ref as R

BF16, F16, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32


def t(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def i(*shape):
    return torch.zeros(shape, dtype=I32)


def rot(q, dim=8, **kw):
    return q.Rotary(dim, device="cpu", **kw)


def rotate(x=None, p=None, r=None, **kw):
    return lambda q: q.rotate(t(2, 3, 16) if x is None else x, i(2) if p is None else p, r or rot(q), **kw)


def append(k=None, v=None, kc=None, vc=None, table=None, lengths=None, rotary=None, **kw):
    def call(q):
        d = lambda x, y: y if x is None else x
        cache = t(4, 16, 2, 32)
        return q.append_kv(d(k, t(3, 2, 32)), d(v, t(3, 2, 32)), d(kc, cache), d(vc, cache.clone()), d(table, i(3, 5)),
                           d(lengths, i(3)), rotary=rotary and rotary(q), **kw)
    return call


def attend(x=None, kc=None, vc=None, table=None, lengths=None, **kw):
    def call(q):
        d = lambda a, b: b if a is None else a
        cache = t(4, 16, 2, 32)
        return q.paged_attention(d(x, t(3, 4, 32)), d(kc, cache), d(vc, cache), d(table, i(3, 5)), d(lengths, i(3)), **kw)
    return call


@pytest.mark.parametrize("call,says", [
    (lambda q: rot(q, 7), "dim must be"), (lambda q: rot(q, 0), "dim must be"), (lambda q: rot(q, 1026), "dim must be"),
    (lambda q: rot(q, layout="other"), "layout"), (lambda q: rot(q, base=1.0), "base"), (lambda q: rot(q, base=math.nan), "base"),
    (lambda q: rot(q, scaling="other"), "scaling is"), (lambda q: rot(q, factor=2.0), "comes with a scaling"),
    (lambda q: rot(q, scaling="linear", factor=0.5), "factor"), (lambda q: rot(q, scaling="linear", factor=math.inf), "factor"),
    (lambda q: rot(q, 2, scaling="base", factor=2.0), "dim >= 4"), (lambda q: rot(q, scaling="parts", factor=2.0), "original_length"),
    (lambda q: rot(q, scaling="parts", factor=2.0, original_length=10, beta_slow=40.0), "beta_slow"),
    (lambda q: rot(q, frequencies=[1.0]), "4 numbers"), (lambda q: rot(q, frequencies=[1.0] * 4, scaling="linear"), "no scaling"),
    (lambda q: rot(q, frequencies=[1.0, 2.0, math.nan, 0.0]), "finite"), (lambda q: rot(q, turn=math.inf), "finite"),
    (rotate(), "device tensors"), (rotate(t(2, 3, 16, dtype=torch.float64)), "x must be"), (rotate(t(16)), "x must be"),
    (rotate(t(2, 3, 1025)), "x must be"), (rotate(t(2, 3, 0)), "x must be"), (rotate(t(2, 3, 6)), "turns 8 elements"),
    (rotate(p=i(3)), "positions"), (rotate(p=t(2, dtype=F32)), "int32 or int64"), (rotate(r=3), "must be a Rotary"),
    (append(), "device tensors"), (append(t(3, 2, 32, dtype=torch.int8)), "k must be"), (append(t(6, 32)), "k must be"),
    (append(v=t(3, 2, 16)), "v must have"), (append(v=t(3, 2, 32, dtype=F16)), "v must have"), (append(kc=t(4, 16, 2, 32, dtype=F32)), "type"),
    (append(kc=t(4, 8, 2, 32)), "both alike"), (append(t(3, 4, 32), t(3, 4, 32)), "do not match"),
    (append(kc=t(4, 16, 1, 32).expand(4, 16, 2, 32)), "must not overlap"), (append(vc=t(1, 16, 2, 32).expand(4, 16, 2, 32)), "must not overlap"),
    (append(kc=t(4, 16, 32, 2).mT, vc=t(4, 16, 32, 2).mT), "contiguous"),
    (append(table=torch.zeros((3, 5), dtype=torch.int64)), "table must be"), (append(table=i(15)), "table must be"),
    (append(lengths=i(4)), "lengths must be"), (append(table=i(2, 5), lengths=i(2)), "need starts"), (append(starts=i(3)), "starts must be"),
    (append(starts=torch.zeros(4, dtype=torch.int64)), "starts must be"), (append(q=t(4, 4, 32)), "q must be"),
    (append(q=t(3, 4, 32, dtype=F16)), "q must be"), (append(rotary=lambda q: rot(q, 64)), "turns 64"),
    (append(positions=i(3)), "need a rotary"), (append(positions=i(4), rotary=rot), "positions"),
    (attend(), "device tensors"), (attend(t(3, 4, 32, dtype=F32)), "q must be"), (attend(t(3, 128)), "q must be"),
    (attend(t(3, 4, 36), t(4, 16, 2, 36), t(4, 16, 2, 36)), "multiple of 8"), (attend(t(3, 4, 264)), "multiple of 8"),
    (attend(t(3, 3, 32)), "cannot share"), (attend(t(3, 130, 32)), "cannot share"), (attend(t(3, 0, 32)), "cannot share"),
    (attend(kc=t(4, 16, 64)), "both alike"), (attend(kc=t(5, 16, 2, 32)), "both alike"), (attend(vc=t(4, 16, 2, 32, dtype=F16)), "type"),
    (attend(window=-1), "window"), (attend(window=1.5), "window"), (attend(window=(1 << 30) + 1), "window"),
    (attend(lengths=torch.zeros(3)), "lengths must be"), (attend(starts=i(3)), "starts must be"),
    (attend(kc=t(4, 16, 2, 36)[..., :32], vc=t(4, 16, 2, 36)[..., :32]), "16-byte aligned"),
    (attend(kc=t(4 * 16 * 64 + 1)[1:].view(4, 16, 2, 32)), "16-byte aligned"),
])
def test_refusals(call, says):
    import qmoe
    with pytest.raises(RuntimeError, match=says):
        call(qmoe)


def test_c_entries_refuse_before_any_launch():
    """(No pointer here is real.)"""
    from qmoe import _lib
    L = _lib.lib()

    def rotate(x=16, type=0, rd=8, inter=0, turn=1.0, T=2, heads=3, D=16, f=16, p=16):
        return L.qmoe_rotate(x, 48, 16, x, 48, 16, type, p, 0, f, rd, inter, turn, T, heads, D, None)
    assert rotate(T=0) == 0 and rotate(heads=0) == 0 and rotate(T=0, f=None, p=None, x=None) == 0
    for kw in (dict(type=3), dict(rd=7), dict(rd=18), dict(rd=-2), dict(inter=2), dict(turn=math.nan), dict(turn=math.inf),
               dict(D=0, rd=0), dict(D=1025), dict(T=-1), dict(heads=-1)):
        assert rotate(**kw) == -1 and rotate(**{"T": 0, **kw}) == -1, kw
    for kw in (dict(x=None), dict(f=None), dict(p=None), dict(T=1 << 30, heads=1 << 20)):
        assert rotate(**kw) == -1, kw

    def append(k=16, q=16, qo=16, type=0, kc=16, table=16, ld=4, width=4, lengths=16, starts=16, f=16, rd=8, T=2, B=2, Hq=4, Hkv=2,
               D=16, page=8, pages=3):
        return L.qmoe_append_kv(k, 32, 16, k, 32, 16, q, 64, 16, qo, type, kc, 256, 32, 16, kc, 256, 32, 16, table, ld, width,
                                lengths, starts, None, 0, f, rd, 0, 1.0, T, B, Hq, Hkv, D, page, pages, None)
    assert append(T=0) == 0
    for kw in (dict(type=5), dict(rd=3), dict(T=-1), dict(B=-1), dict(Hkv=0), dict(Hq=-1), dict(page=0), dict(page=(1 << 30) + 1),
               dict(pages=-1), dict(width=-1), dict(ld=-1), dict(B=3, starts=None), dict(q=None), dict(qo=None), dict(Hq=0),
               dict(Hq=1 << 20), dict(D=2000)):
        assert append(**kw) == -1 and append(**{"T": 0, **kw}) == -1, kw
    for kw in (dict(k=None), dict(kc=None), dict(table=None), dict(lengths=None), dict(f=None)):
        assert append(**kw) == -1, kw

    def attend(q=16, kc=16, k_slot=64, type=0, table=16, ld=4, width=4, lengths=16, starts=16, out=16, T=2, B=2, Hq=4, Hkv=2, D=32,
               page=8, pages=3, scale=1.0, window=0, ws=None, nbytes=0):
        return L.qmoe_paged_attention(q, 128, 32, kc, 512, k_slot, 32, kc, 512, 64, 32, type, table, ld, width, lengths, starts, out,
                                      T, B, Hq, Hkv, D, page, pages, scale, window, ws, nbytes, None)
    assert attend(T=0) == 0
    for kw in (dict(type=2), dict(T=-1), dict(B=-1), dict(Hq=3), dict(Hq=0), dict(Hkv=0), dict(Hq=130, Hkv=2), dict(D=36), dict(D=264),
               dict(D=0), dict(page=0), dict(pages=-1), dict(scale=math.inf), dict(window=-1), dict(k_slot=60), dict(kc=8),
               dict(B=3, starts=None), dict(width=-1), dict(ld=-1), dict(Hq=8192, Hkv=4096),
               dict(window=(1 << 30) + 1), dict(width=1 << 20, page=1 << 11), dict(k_slot=1 << 28), dict(k_slot=-64),
               dict(B=1 << 20, Hkv=4, width=1 << 20, page=16)):
        assert attend(**kw) == -1 and attend(**{"T": 0, **kw}) == -1, kw
    for kw in (dict(q=None), dict(kc=None), dict(table=None), dict(lengths=None), dict(out=None), dict(T=1 << 30, Hq=4)):
        assert attend(**kw) == -1, kw


def test_cache_places_apart():
    from qmoe.rotary import _apart
    for sizes, steps, width, fine in (((4, 16, 2), (1024, 64, 32), 32, True), ((4, 2, 16), (1024, 512, 32), 32, True),
                                      ((4, 16, 2), (1024, 32, 512), 32, True), ((4, 16, 2), (1000, 64, 32), 32, False),
                                      ((4, 16, 2), (1024, 64, 16), 32, False), ((4, 1, 2), (64, 0, 32), 32, True),
                                      ((2, 2), (32, 32), 32, False), ((2, 2), (0, 32), 32, False), ((1, 1), (0, 0), 8, True)):
        assert _apart(sizes, steps, width) is fine, (sizes, steps)


def test_frequencies():
    """Fractions of a turn of 64 bits, signed in memory, against the angle in whole numbers."""
    from qmoe import Rotary
    for dim, base, kw in ((128, 1.0e4, {}), (64, 1.0e6, dict(scaling="base", factor=4.0)),
                          (96, 5.0e5, dict(scaling="parts", factor=8.0, original_length=8192))):
        r = Rotary(dim, base, device="cpu", **kw)
        f, turn = A.frequencies(dim, base, kw.get("scaling"), kw.get("factor", 1.0), kw.get("original_length"))
        got = r.frequencies.double() * 2.0 ** -64
        # whole multiples of 2^-64, so off by half of one beside the 64-bit powers' own error
        assert torch.allclose(got, f / (2 * math.pi), rtol=1e-14, atol=2.0 ** -64) and r.turn == pytest.approx(turn, rel=1e-15)
    r = Rotary(6, frequencies=[-1.0, 4.0, 2 * math.pi * 3], device="cpu")
    got = [v % 2 ** 64 / 2 ** 64 for v in r.frequencies.tolist()]
    assert got[0] == pytest.approx(1 - 1 / (2 * math.pi)) and got[1] == pytest.approx(4 / (2 * math.pi)) and got[2] == 0
    # in "parts" the fastest pair stays and the slowest is divided
    f = Rotary(128, 1.0e4, scaling="parts", factor=4.0, original_length=4096, device="cpu").frequencies.double()
    plain = Rotary(128, 1.0e4, device="cpu").frequencies.double()
    assert f[0] == plain[0] and f[-1] / plain[-1] == pytest.approx(0.25) and (f.diff() < 0).all()


def test_references():
    """The references against torch's own functions and values worked out by hand."""
    x = torch.tensor([[[1.0, 0.0, 5.0]]])
    p = torch.tensor([1])
    f = torch.tensor([math.pi / 2], dtype=torch.float64)
    assert torch.allclose(A.rotate(x, p, f, 2.0, "half")[0], torch.tensor([[[0.0, 2.0, 5.0]]], dtype=torch.float64))
    x = torch.arange(8.0).view(1, 1, 8)
    for layout, pairs in (("half", ((0, 4), (1, 5), (2, 6), (3, 7))), ("interleaved", ((0, 1), (2, 3), (4, 5), (6, 7)))):
        f, _ = A.frequencies(8, 100.0)
        out = A.rotate(x, torch.tensor([3]), f, 1.0, layout)[0].view(8)
        for n, (a, b) in enumerate(pairs):
            z = complex(float(a), float(b)) * complex(math.cos(3 * 100.0 ** (-n / 4)), math.sin(3 * 100.0 ** (-n / 4)))
            assert out[a] == pytest.approx(z.real) and out[b] == pytest.approx(z.imag)
    g = torch.Generator().manual_seed(1)
    page, D, n, L = 4, 16, 5, 23
    caches = [torch.randn((7, page, 2, D), generator=g).to(BF16) for _ in range(2)]
    table = torch.randperm(7, generator=g)[None, :6].int()
    q = torch.randn((n, 4, D), generator=g).to(BF16)
    k, v = (c[table[0].long()].flatten(0, 1)[:L].double().repeat_interleave(2, 1).transpose(0, 1) for c in caches)
    mask = torch.ones(n, L, dtype=torch.bool).tril(L - n)
    want = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(0, 1), k, v, attn_mask=mask).transpose(0, 1)
    lengths, starts = torch.tensor([L]), torch.tensor([0, n])
    out, bound = A.attention(q, *caches, table, lengths, starts)
    assert torch.allclose(out, want) and (bound < 0.05).all()
    mask &= ~torch.ones(n, L, dtype=torch.bool).tril(L - n - 6)
    want = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(0, 1), k, v, attn_mask=mask).transpose(0, 1)
    assert torch.allclose(A.attention(q, *caches, table, lengths, starts, window=6)[0], want)
    table[0, :5] = -1
    out = A.attention(q, *caches, table, lengths, starts)[0]
    assert not out[0].any() and not out[1].any() and out[2:].any(2).all()  # places 20, 21, 22 are left


def test_planted_mistakes_are_seen():
    """One key too many or too few, a page mistaken, a head of another group: beyond the bound."""
    g = torch.Generator().manual_seed(2)
    page, D, L = 16, 64, 300
    caches = [torch.randn((25, page, 2, D), generator=g).to(BF16) for _ in range(2)]
    table = torch.randperm(25, generator=g)[None, :19].int()
    q = (torch.randn((3, 4, D), generator=g) * 2).to(BF16)
    lengths, starts = torch.tensor([L]), torch.tensor([0, 3])
    want, bound = A.attention(q, *caches, table, lengths, starts)
    R.assert_close(want.to(BF16), want, bound, "same")
    swapped = table.clone()
    swapped[0, [3, 4]] = table[0, [4, 3]]
    R.assert_close(A.attention(q, *caches, swapped, lengths, starts)[0].to(BF16), want, bound, "whole pages may change places")
    swapped[0, 3] = table[0, 7]
    wrong = [A.attention(q, *caches, table, lengths - 1, starts)[0], A.attention(q, *caches, table, lengths, starts, window=290)[0],
             A.attention(q, *caches, swapped, lengths, starts)[0],
             A.attention(q, *[c.flip(2) for c in caches], table, lengths, starts)[0],
             A.attention(q, *caches, table, lengths, starts, scale=0.126)[0]]
    for w in wrong:
        with pytest.raises(AssertionError):
            R.assert_close(w.to(BF16), want, bound, "planted")


def test_grid_fits_32_bits():
    """A grid holds fewer than 2^32 threads: the C entry refuses more (a call that it takes asks for its workspace,
    before any launch)."""
    from qmoe import _lib

    def attend(T, B, Hq, Hkv):
        return _lib.lib().qmoe_paged_attention(16, 8 * Hq, 8, 16, 16 * 8 * Hkv, 8 * Hkv, 8, 16, 16 * 8 * Hkv, 8 * Hkv, 8, 0, 16, 4, 4, 16, 16,
                                               16, T, B, Hq, Hkv, 8, 16, 3, 1.0, 0, None, 0, None)
    assert attend(1 << 24, 2, 64, 64) == -2 and attend((1 << 25) - 1, 2, 64, 64) == -1
    assert attend(1 << 22, 1 << 16, 64, 64) == -2 and attend(1 << 24, 1 << 18, 64, 64) == -1


def test_list_of_few_rows_fits_32_bits():
    """Places of the list of single tokens' keys, with the up to 768 that equal shares are rounded up by, stay below
    2^31: the C entry refuses more (a call that it takes asks for its workspace, before any launch)."""
    from qmoe import _lib

    def attend(B, tiles):  # tiles of 128 keys that a table names, two places a head beside them, and one more tile
        return _lib.lib().qmoe_paged_attention(16, 128, 32, 16, 128 * 32, 32, 32, 16, 128 * 32, 32, 32, 0, 16, tiles, tiles, 16, None,
                                               16, B, B, 1, 1, 32, 128, 3, 1.0, 0, None, 0, None)
    most = 2 ** 31 - 1 - 768
    B = 256
    fits = most // B - 3
    assert B * (fits + 1 + 3) <= 0x7fffff00  # within a rounder limit
    assert attend(B, fits) == -2 and attend(B, fits + 1) == -1
    assert attend(1 << 22, 1) == -2 and attend(1 << 22, 512) == -1


def test_list_of_few_rows_past_64_bits():
    """A batch whose places pass 64 bits is refused like any other that is too long."""
    from qmoe import _lib

    def attend(B, page):
        return _lib.lib().qmoe_paged_attention(16, 4096 * 8, 8, 16, 4096 * 8, 0, 8, 16, 4096 * 8, 0, 8, 0, 16, 1, 1, 16, 16, 16, 1, B,
                                               4096, 4096, 8, page, 3, 1.0, 0, None, 0, None)
    assert attend(1 << 16, 16) == -2 and attend(1 << 28, 1 << 30) == -1 and attend((1 << 31) - 1, 1 << 30) == -1
