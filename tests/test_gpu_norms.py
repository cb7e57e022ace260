"""block_norm and block_residual against the formulas in 64 bits."""
import pytest
import torch

import operators_ref as R

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def log(msg):
    print(f"[case] {msg}", flush=True)


def gen(device, seed):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return lambda *shape, std=1.0, dtype=BF16: (torch.randn(shape, generator=g, device=device) * std).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", [(1, 1), (3, 2), (1, 7), (5, 8), (2, 63), (1, 64), (7, 255), (2, 512), (3, 513), (1, 2048),
                                 (4, 2560), (129, 1111), (1030, 640), (2, 4095), (300, 4096), (3, 8192), (2, 8195),
                                 (1, 16384), (2, 32767), (1, 32768)])
@pytest.mark.parametrize("xt,ot,wt,offset", [(BF16, BF16, BF16, 0.0), (F16, F16, F32, 1.0), (F32, F32, F32, 0.0),
                                             (F32, BF16, BF16, 1.0), (F32, F16, F16, 0.0)])
def test_block_norm(device, T, H, xt, ot, wt, offset):
    from qmoe import block_norm
    log(f"block_norm T={T} H={H} {xt} {ot}")
    n = gen(device, T * 7 + H)
    x, w = n(T, H, std=3.0, dtype=xt), n(H, std=0.3, dtype=wt)
    out = block_norm(x, w, offset=offset, out_dtype=ot)
    assert out.dtype == ot and out.is_contiguous()
    R.assert_close(out, *R.block_norm(x, w, 1e-6, offset, ot), "block_norm")


# more rows than workgroups stay resident: one wave a row, several, sixteen; short, odd, even
MANY = [(20001, 64), (9001, 641), (5000, 1024), (5003, 1033), (3001, 2560), (1300, 4096), (1100, 8192), (601, 9001),
        (800, 16384), (530, 16390)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", MANY)
@pytest.mark.parametrize("xt,ot", [(BF16, BF16), (F32, F32), (F32, F16)])
def test_block_norm_many_rows(device, T, H, xt, ot):
    from qmoe import block_norm
    log(f"block_norm T={T} H={H} {xt} {ot}")
    n = gen(device, T + H)
    x, w = n(T, H, std=3.0, dtype=xt), n(H, std=0.3)
    x[T // 2, H // 2] = torch.finfo(xt).max  # this row's squares leave the fp32 range, the others' not
    R.assert_close(block_norm(x, w, out_dtype=ot), *R.block_norm(x, w, 1e-6, 0.0, ot), "block_norm")


@pytest.mark.gpu
@pytest.mark.parametrize("xt", [BF16, F32])
def test_block_norm_layouts(device, xt):
    """Rows apart, off any alignment, shared rows, columns apart, more dimensions, a sliced weight."""
    from qmoe import block_norm
    n = gen(device, 5)
    wide, w = n(9, 700, dtype=xt), n(1400)[1::2]
    views = [wide[:, :512], wide[:, 3:516], wide[:, 1:600], wide[::2, 5:70], wide[:1].expand(6, 700), wide.t(),
             wide.view(3, 3, 700), wide.view(9, 7, 100).transpose(0, 1), wide[0, :33], wide[4]]
    for i, x in enumerate(views):
        log(f"layout {i} {tuple(x.shape)} {x.stride()}")
        before = wide.clone()
        out = block_norm(x, w[:x.shape[-1]])
        assert out.shape == x.shape
        R.assert_close(out, *R.block_norm(x, w[:x.shape[-1]]), f"layout {i}")
        assert torch.equal(wide, before)
    for shape in ((0, 16), (3, 0, 16)):
        assert block_norm(torch.empty(shape, dtype=xt, device=device), n(16)).shape == shape


@pytest.mark.gpu
@pytest.mark.parametrize("xt,ot", [(BF16, BF16), (F16, F16), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("H", [64, 1000, 2560])
def test_block_norm_values(device, xt, ot, H):
    """Zeros, the type's largest and smallest values, rows whose squares leave the fp32 range,
    infinities and NaN in one row only."""
    from qmoe import block_norm
    log(f"values H={H} {xt}")
    n = gen(device, H)
    f = torch.finfo(xt)
    x = n(12, H, dtype=xt)
    x[0] = 0
    x[1] = f.max
    x[2] = f.max
    x[2, ::2] = -f.max
    x[3] = f.smallest_normal
    x[4] = (x[4].float() * (f.max / 8)).to(xt)
    x[5, 3] = f.max
    x[6, H - 1] = float("nan")
    x[7, 0] = float("inf")
    x[8, 1] = -float("inf")
    x[9] = x[9] * 1e-4
    w = n(H, dtype=F32)
    for eps in (1e-6, 1e-12, 1.0):
        out = block_norm(x, w, eps=eps, out_dtype=ot)
        exact, bound = R.block_norm(x, w, eps, 0.0, ot)
        # a row with an infinity: inf / inf at its place, finite / inf elsewhere (-0 and 0 alike)
        R.assert_close(out, exact, bound, f"values eps={eps}")


COMBOS = [  # y, residual, weights, post, gate shape, gate type, act, scale, next, offset
    (BF16, BF16, BF16, True, "row", BF16, "sigmoid", 1.0, True, 0.0),
    (BF16, BF16, BF16, False, None, None, None, 1.0, True, 0.0),
    (BF16, BF16, F32, False, None, None, None, 0.22, False, 0.0),
    (BF16, F32, F32, False, "channel", BF16, None, 0.22, True, 1.0),
    (BF16, F32, BF16, True, "full", F32, "sigmoid", -1.5, True, 1.0),
    (F16, F16, F16, True, "full", F16, "sigmoid", 0.5, False, 0.0),
    (F16, F32, F32, True, "row", F32, None, 1.0, True, 0.0),
    (F32, F32, F32, True, "channel", F32, "sigmoid", 1.0, True, 1.0),
    (F32, F32, BF16, True, "one", F16, "sigmoid", 0.0, True, 0.0),
]


def operands(n, T, H, c):
    yt, rt, wt, post, gshape, gt, act, scale, nxt, offset = c
    shape = {None: None, "row": (T, 1), "channel": (H,), "full": (T, H), "one": (1, 1)}[gshape]
    kw = dict(post_weight=n(H, std=0.3, dtype=wt) if post else None, scale=scale, offset=offset, gate_act=act,
              gate=None if shape is None else n(*shape, std=2.0, dtype=gt),
              next_weight=n(H, std=0.3, dtype=wt) if nxt else None)
    return n(T, H, std=0.5, dtype=yt), n(T, H, std=3.0, dtype=rt), kw


def check_residual(got, exact, what):
    got = got if isinstance(got, tuple) else (got,)
    assert len(got) == len(exact)
    for g, e, name in zip(got, exact, ("h", "x")):
        R.assert_close(g, *e, f"{what} {name}")


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", [(1, 1), (2, 9), (1, 64), (3, 515), (1, 2048), (4, 2560), (700, 2560), (65, 2047),
                                 (300, 4096), (2, 8192), (3, 16384), (2, 20001), (1, 32768)])
@pytest.mark.parametrize("c", COMBOS)
def test_block_residual(device, T, H, c):
    from qmoe import block_residual
    log(f"block_residual T={T} H={H} {c}")
    y, r, kw = operands(gen(device, T + 3 * H), T, H, c)
    keep = y.clone(), r.clone()
    got = block_residual(y, r, **kw)
    check_residual(got, R.block_residual(y, r, **kw), "block_residual")
    assert torch.equal(y, keep[0]) and torch.equal(r, keep[1])
    # in place: the same bits, over the residual, whose version moves on
    v = r._version
    again = block_residual(y, r, inplace=True, **kw)
    h = again[0] if isinstance(again, tuple) else again
    assert h is r and r._version > v
    for a, b in zip(got if isinstance(got, tuple) else (got,), again if isinstance(again, tuple) else (again,)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", MANY)
@pytest.mark.parametrize("c", [COMBOS[0], COMBOS[3], COMBOS[5], COMBOS[6], COMBOS[7]])
def test_block_residual_many_rows(device, T, H, c):
    from qmoe import block_residual
    log(f"block_residual T={T} H={H} {c}")
    y, r, kw = operands(gen(device, T + 5 * H), T, H, c)
    want = R.block_residual(y, r, **kw)
    got = block_residual(y, r, **kw)
    check_residual(got, want, "block_residual")
    again = block_residual(y, r, inplace=True, **kw)
    for a, b in zip(got if isinstance(got, tuple) else (got,), again if isinstance(again, tuple) else (again,)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("c", [COMBOS[0], COMBOS[4], COMBOS[5]])
def test_block_residual_layouts(device, c):
    """Strided and shared operands, more dimensions, a residual updated in place between rows of
    its neighbours, and the block output being the residual itself."""
    from qmoe import block_residual
    log(f"layouts {c}")
    n = gen(device, 3)
    T, H = 10, 333
    _, _, kw = operands(n, T, H, c)
    wide_y, wide_r = n(T, H + 5, dtype=c[0]), n(T, H + 3, dtype=c[1])
    y, r = wide_y[:, 5:], wide_r[:, 1:H + 1]
    check_residual(block_residual(y, r, **kw), R.block_residual(y, r, **kw), "strided")
    y1 = wide_y[:1, :H].expand(T, H)
    check_residual(block_residual(y1, r, **kw), R.block_residual(y1, r, **kw), "shared rows")
    if c[4] != "row":
        kw3 = {**kw, "gate": None, "gate_act": None}
    else:
        kw3 = {**kw, "gate": kw["gate"].view(2, 5, 1)}
    y3, r3 = y.reshape(2, 5, H), r.reshape(2, 5, H)
    got = block_residual(y3, r3, **kw3)
    flat = {**kw3, "gate": None if kw3["gate"] is None else kw3["gate"].view(T, 1)}
    want = [(e.view(2, 5, H), b.view(2, 5, H)) for e, b in R.block_residual(y, r, **flat)]
    check_residual(got, want, "three dimensions")
    before = wide_r.clone()
    want = R.block_residual(y, r, **kw)
    check_residual(block_residual(y, r, inplace=True, **kw), want, "in place, strided")
    assert torch.equal(wide_r[:, 0], before[:, 0]) and torch.equal(wide_r[:, H + 1:], before[:, H + 1:])
    if c[0] == c[1]:
        z = n(T, H, dtype=c[0])
        want = R.block_residual(z, z, **kw)
        check_residual(block_residual(z, z, inplace=True, **kw), want, "itself")
    with pytest.raises(RuntimeError, match="overlaps"):
        block_residual(wide_r[:, :H], wide_r[:, 1:H + 1], inplace=True) if c[0] == c[1] else block_residual(
            y, r, gate=wide_r[:, :H], inplace=True)


@pytest.mark.gpu
def test_block_residual_extremes(device):
    """Rows with infinities and NaN leave the other rows alone; saturated gates; squares
    beyond the fp32 range in y and in h."""
    from qmoe import block_residual
    n = gen(device, 11)
    H = 1500
    for yt, rt in ((BF16, BF16), (F32, F32), (BF16, F32)):
        log(f"extremes {yt} {rt}")
        y, r = n(8, H, dtype=yt), n(8, H, dtype=rt)
        gate = n(8, H, dtype=yt)
        gate[0, :4] = torch.tensor([200.0, -200.0, 0.0, -80.0], device=device)
        y[1] = torch.finfo(yt).max
        r[2] = 1e30
        y[3, 5] = float("nan")
        r[4, 6] = float("inf")
        y[5] = 0
        r[5] = 0
        gate[6, 2] = float("inf")
        gate[7, 2] = -float("inf")
        kw = dict(post_weight=n(H), gate=gate, gate_act="sigmoid", next_weight=n(H))
        check_residual(block_residual(y, r, **kw), R.block_residual(y, r, **kw), "extremes")


@pytest.mark.gpu
def test_next_norm_is_block_norm(device):
    """The next block's input is block_norm of the sum, where the stream holds it unrounded."""
    from qmoe import block_norm, block_residual
    n = gen(device, 21)
    y, r, w = n(77, 2560), n(77, 2560, dtype=F32), n(2560)
    h, x = block_residual(y, r, next_weight=w)
    assert torch.equal(x, block_norm(h, w, out_dtype=BF16))


@pytest.mark.gpu
def test_inplace_beside_its_operands(device):
    """y, the residual and a gate as columns of one tensor."""
    from qmoe import block_residual
    n = gen(device, 31)
    wide = n(700, 1025 + 2 * 512)
    y, r, gate = wide[:, :512], wide[:, 512:1024], wide[:, 1024:1025]
    keep, want = wide.clone(), R.block_residual(y, r, gate=gate, gate_act="sigmoid")
    check_residual(block_residual(y, r, gate=gate, gate_act="sigmoid", inplace=True), want, "beside")
    assert torch.equal(wide[:, :512], keep[:, :512]) and torch.equal(wide[:, 1024:], keep[:, 1024:])


@pytest.mark.gpu
def test_other_device(device, monkeypatch):
    """Tensors of a device that is not the current one: the call is made again with it current."""
    from qmoe import _lib, block_norm, block_residual, token_logprobs
    n = gen(device, 41)
    x, w = n(5, 640), n(640)
    tok = torch.zeros(5, dtype=torch.int64, device=device)
    calls = (lambda: block_norm(x, w, offset=1.0), lambda: block_residual(x, x, post_weight=w, scale=0.5, next_weight=w),
             lambda: token_logprobs(x, tok, top=3))
    want = [c() for c in calls]
    current = _lib.current_device
    for c, e in zip(calls, want):
        answers = iter([1])
        monkeypatch.setattr(_lib, "current_device", lambda: next(answers, current()))
        got = c()
        assert next(answers, None) is None
        for a, b in zip(got if isinstance(got, tuple) else (got,), e if isinstance(e, tuple) else (e,)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_norms_with_gradients(device):
    from qmoe import block_norm, block_residual
    w = torch.ones(16, device=device, requires_grad=True)
    x = torch.ones((2, 16), device=device)
    with pytest.raises(RuntimeError, match="no backward pass"):
        block_norm(x, w)
    with pytest.raises(RuntimeError, match="no backward pass"):
        block_residual(x, x, next_weight=w)
    with torch.no_grad():
        assert block_norm(x, w).shape == x.shape
    with torch.inference_mode():
        r = x.clone()
        assert block_residual(x, r, inplace=True) is r


@pytest.mark.gpu
def test_negated_views(device):
    """Imaginary parts of conjugates, whose memory holds the other sign, as every operand that can be one."""
    from qmoe import block_norm, block_residual, token_logprobs
    n = gen(device, 51)

    def view(*shape):
        v = torch.imag(torch.complex(n(*shape, dtype=F32), n(*shape, dtype=F32)).conj())
        assert v.is_neg()
        return v
    for T, H in ((5, 1), (1, 1), (4, 77)):
        log(f"negated T={T} H={H}")
        x, w, y, r, gate = view(T, H), view(H), view(T, H), view(T, H), view(T, 1)
        R.assert_close(block_norm(x, w), *R.block_norm(x, w), "block_norm")
        kw = dict(post_weight=w, gate=gate, scale=0.5, next_weight=w)
        check_residual(block_residual(y, r, **kw), R.block_residual(y, r, **kw), "block_residual")
        wide = gate.expand(T, H)
        check_residual(block_residual(y, r, gate=wide), R.block_residual(y, r, gate=wide), "expanded gate")
        with pytest.raises(RuntimeError, match="negated"):
            block_residual(y, r, inplace=True)
        keep = y.clone()
        plain = r.clone().resolve_neg()
        want = R.block_residual(y, plain, gate=gate)
        check_residual(block_residual(y, plain, gate=gate, inplace=True), want, "in place")
        assert torch.equal(y, keep)
        got, want = token_logprobs(x, top=3), R.token_logprobs(x, top=3)
        assert torch.equal(got.top_ids, want[2])
        R.assert_close(got.entropy, *want[1], "entropy")
        R.assert_close(got.top_logprobs, *want[3], "top_logprobs")


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,H", [(3, 5, 333), (1, 4, 64), (4, 1, 64), (2, 3, 1), (70, 11, 2560)])
def test_gates_per_sequence(device, B, S, H):
    """Gates of a batch of sequences: one value for each of them, each and channel, each position of
    all, each channel, one in all."""
    from qmoe import block_residual
    n = gen(device, B * S + H)
    y, r, w = n(B, S, H), n(B, S, H, dtype=F32), n(H)
    for shape in ((B, 1, 1), (B, 1, H), (1, S, 1), (S, 1), (1, S, H), (1, 1, H), (H,), (1,), ()):
        log(f"gate {shape} of {(B, S, H)}")
        gate = n(*shape)
        for act in (None, "sigmoid"):
            want = R.block_residual(y, r, gate=gate, gate_act=act, next_weight=w)
            check_residual(block_residual(y, r, gate=gate, gate_act=act, next_weight=w), want, f"gate {shape}")
