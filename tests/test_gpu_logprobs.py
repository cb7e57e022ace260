"""token_logprobs against the formulas in 64 bits, and the operators in use together."""
import pytest
import torch

import operators_ref as R

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def log(msg):
    print(f"[case] {msg}", flush=True)


def gen(device, seed):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def rows(g, T, V, dtype, std=2.5):
    x = torch.randn((T, V), generator=g, device=g.device) * std
    hot = torch.randint(0, V, (T, min(V, 8)), generator=g, device=g.device)
    return x.scatter_add_(1, hot, 4 + 8 * torch.rand(hot.shape, generator=g, device=g.device)).to(dtype)


def check(logits, tokens=None, top=0, allowed=None):
    from qmoe import token_logprobs
    got = token_logprobs(logits, tokens, top=top, allowed=allowed)
    want = R.token_logprobs(logits, tokens, top, allowed)
    for g, w, name in zip((got.logprobs, got.entropy, got.top_logprobs), (want[0], want[1], want[3]),
                          ("logprobs", "entropy", "top_logprobs")):
        assert (g is None) == (w is None), name
        if g is not None:
            assert g.dtype == F32 and g.is_contiguous()
            R.assert_close(g, *w, name)
    if top:
        assert got.top_ids.dtype == torch.int64
        assert torch.equal(got.top_ids, want[2]), "top_ids"
    else:
        assert got.top_ids is None and want[2] is None
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,V,m,top", [(1, 1, 1, 3), (3, 2, 2, 2), (1, 31, 1, 32), (5, 63, 1, 32), (2, 64, 1, 20),
                                       (4, 257, 3, 1), (1, 2047, 1, 20), (2, 8192, 1, 32), (1, 8193, 1, 5),
                                       (300, 1000, 1, 8), (7, 50003, 4, 20), (1, 131072, 1, 20), (33, 131072, 1, 0),
                                       (1, 262147, 1, 32), (1200, 4099, 1, 20), (600, 20001, 0, 5), (2, 1000003, 1, 20),
                                       (100, 60000, 1, 32), (400, 33011, 1, 20), (1023, 17000, 1, 5), (511, 40000, 2, 0),
                                       (3, 32768, 1, 20), (3, 32769, 1, 20), (3, 32776, 1, 20), (5, 16391, 1, 20),
                                       (48, 70001, 1100, 8), (1100000, 9, 1, 3),
                                       # whole rows on 16, 8 and 4 waves, one and more steps, ends on and off them
                                       (200, 131072, 1, 20), (161, 140001, 1, 32), (64, 65543, 3, 5), (256, 32768, 1, 20),
                                       (257, 32768, 1, 20), (500, 16384, 1, 32), (500, 16383, 1, 5), (9, 4096, 1, 20),
                                       (9, 4104, 1, 20), (9, 8193, 1, 32), (1100, 33000, 1, 0), (1100, 33000, 1, 2),
                                       (513, 40000, 1, 20), (127, 131077, 1, 20), (70, 80000, 1, 7)])
def test_token_logprobs(device, T, V, m, top, dtype):
    log(f"token_logprobs T={T} V={V} m={m} top={top} {dtype}")
    g = gen(device, T + V)
    x = rows(g, T, V, dtype)
    tokens = torch.randint(0, V, (T, m), generator=g, device=device) if m != 1 else \
        torch.randint(0, V, (T,), generator=g, device=device)
    check(x, tokens if m else None, top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,V", [(1, 100), (9, 3001), (3, 131072), (700, 9000), (100, 40001), (300, 20000)])
def test_allowed(device, T, V, dtype):
    """Masks by row and for all rows, whatever the masked places hold; rows with one token left and
    with none."""
    log(f"allowed T={T} V={V} {dtype}")
    g = gen(device, V)
    x = rows(g, T, V, dtype)
    tokens = torch.randint(0, V, (T, 2), generator=g, device=device)
    for share in (0.5, 0.01):
        allowed = torch.rand((T, V), generator=g, device=device) < share
        if T > 2:
            allowed[1] = False
            allowed[2] = False
            allowed[2, V - 1] = True
        junk = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).max, torch.finfo(dtype).min],
                            device=device)[torch.randint(0, 5, (T, V), generator=g, device=device)].to(dtype)
        check(torch.where(allowed, x, junk), tokens, 20, allowed)
        one = allowed[0].clone()
        check(torch.where(one, x, junk), tokens, 20, one)
        check(torch.where(one, x, junk), tokens, 4, one.expand(T, V))
    # any byte but 0 allows, in a mask made of bytes
    some = torch.randint(0, 3, (V,), generator=g, device=device) * 127
    some = torch.where(some == 254, 255, some).to(torch.uint8)
    check(x, tokens, 5, some.ne(0))
    from qmoe import token_logprobs
    for a, b in zip(token_logprobs(x, tokens, top=5, allowed=some.view(torch.bool)),
                    token_logprobs(x, tokens, top=5, allowed=some.ne(0))):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("V", [50, 5000, 70001])
def test_values(device, V, dtype):
    """Equal logits, sorted ones, -inf, the type's extremes, NaN and +inf; zeros of both signs; one
    token that takes everything."""
    log(f"values V={V} {dtype}")
    g = gen(device, V)
    f = torch.finfo(dtype)
    x = rows(g, 16, V, dtype)
    x[0] = 0
    x[1] = 3.5
    x[2] = torch.sort(x[2].float())[0].to(dtype)
    x[3] = torch.sort(x[3].float(), descending=True)[0].to(dtype)
    x[4] = -float("inf")
    x[5, :V - 3] = -float("inf")
    x[6, V // 2] = float("nan")
    x[7, V - 1] = float("inf")
    x[8] = f.min
    x[9] = f.max
    x[10] = f.min
    x[10, 7] = 2.0
    x[11, ::3] = f.min
    x[12] = 0
    x[12, ::2] = -0.0
    x[12, 5] = -1.0
    x[13, 11] = 60.0
    x[14] = x[14] / 64
    x[15] = (x[15].float() * 0 + torch.arange(V, device=device) // 40).clamp(max=2000).to(dtype)
    tokens = torch.randint(0, V, (16, 3), generator=g, device=device)
    tokens[:, 0] = 7
    got = check(x, tokens, 32)
    assert got.logprobs[4].eq(-float("inf")).all() and got.entropy[4] == 0 and got.top_ids[4].eq(-1).all()
    for bad in (6, 7):
        assert got.logprobs[bad].isnan().all() and got.entropy[bad].isnan() and got.top_logprobs[bad].isnan().all()
        assert got.top_ids[bad].eq(-1).all()
    one = got.logprobs[10, 0]
    assert one == 0 and got.entropy[10] == 0


@pytest.mark.gpu
def test_tokens_out_of_range(device):
    g = gen(device, 1)
    x = rows(g, 6, 500, BF16)
    tokens = torch.tensor([-1, -100, 500, 1 << 40, 499, -(1 << 40)], device=device)
    got = check(x, tokens, 0)
    assert got.logprobs[[0, 1, 5]].eq(0).all() and got.logprobs[[2, 3]].isnan().all()
    x[0, 3] = float("nan")  # padding scores nothing in any row
    assert check(x, tokens, 2).logprobs[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layouts(device, dtype):
    """A slice of a padded vocabulary, rows off any alignment, shared rows, columns apart, other
    dimensions, empty batches."""
    from qmoe import token_logprobs
    g = gen(device, 2)
    wide = rows(g, 12, 3003, dtype)
    mask = torch.rand((12, 3003), generator=g, device=device) < 0.7
    tok = torch.randint(0, 60, (12,), generator=g, device=device)
    for i, f in enumerate([lambda a: a[:, :3000], lambda a: a[:, 3:], lambda a: a[::2, 1:2002], lambda a: a[:1].expand(5, 3003),
                           lambda a: a[:, ::3], lambda a: a.t()[:100], lambda a: a[:, 7:71]]):
        x, ok = f(wide), f(mask)
        log(f"layout {i} {tuple(x.shape)} {x.stride()}")
        t = tok[:1].expand(x.shape[0]) % x.shape[1]
        check(x, t, 5)
        check(x, t, 5, ok)
        check(x, t, 5, ok[0])
    x3, t3 = wide.view(3, 4, 3003), tok.view(3, 4)
    got = check(x3, t3, 6, mask.view(3, 4, 3003))
    assert got.top_ids.shape == (3, 4, 6) and got.entropy.shape == (3, 4)
    check(x3, t3[..., None].expand(3, 4, 2), 0)
    got = check(wide[0], tok[0], 3)
    assert got.logprobs.shape == () and got.top_ids.shape == (3,)
    check(wide[0], tok, 0)
    for lead in ((0,), (2, 0)):
        r = token_logprobs(torch.empty((*lead, 10), dtype=dtype, device=device),
                           torch.empty((*lead, 3), dtype=torch.int64, device=device), top=4)
        assert r.logprobs.shape == (*lead, 3) and r.entropy.shape == lead and r.top_ids.shape == (*lead, 4)
    r = token_logprobs(wide, torch.empty((12, 0), dtype=torch.int64, device=device))
    assert r.logprobs.shape == (12, 0)


@pytest.mark.gpu
def test_same_bits_again(device):
    """No result depends on the order in which workgroups finish."""
    from qmoe import token_logprobs
    g = gen(device, 4)
    for T, V in ((1, 131072), (40, 70001), (3, 5000)):
        log(f"again T={T} V={V}")
        x = rows(g, T, V, BF16)
        tok = torch.randint(0, V, (T,), generator=g, device=device)
        first = token_logprobs(x, tok, top=20)
        for _ in range(20):
            assert all(torch.equal(a, b) for a, b in zip(first, token_logprobs(x, tok, top=20)))


@pytest.mark.gpu
def test_longest_row(device):
    """2^30 logits in one row, the most that is taken: all equal but a few."""
    import math
    from qmoe import token_logprobs
    V = 1 << 30
    log("longest row")
    x = torch.zeros(V, dtype=BF16, device=device)
    at = [V - 1, 0, V // 2 + 3, 77777, V - 9]
    for i, v in enumerate(at):
        x[v] = 9.0 - i
    z = V - len(at) + sum(math.exp(9.0 - i) for i in range(len(at)))
    got = token_logprobs(x, torch.tensor([5, V - 1], device=device), top=7)
    first = [v for v in range(2, 10) if v not in at][:2]
    # a lane adds its 65536 equal terms in steps of 32: 32 + 2048 additions, then the tree
    tol = (32 + 2048 + 64) * R.U + 2 * R.U * math.log(z)
    assert got.top_ids.tolist() == at + [1, 2] == at + [1] + first[:1]
    want = [9.0 - i - math.log(z) for i in range(len(at))] + [-math.log(z)] * 2
    assert all(abs(a - b) <= tol for a, b in zip(got.top_logprobs.tolist(), want))
    assert abs(got.logprobs[0].item() + math.log(z)) <= tol and abs(got.logprobs[1].item() - want[0]) <= tol
    ent = math.log(z) - sum(math.exp(9.0 - i) * (9.0 - i) for i in range(len(at))) / z
    assert abs(got.entropy.item() - ent) <= tol * (1 + math.log(z))


@pytest.mark.gpu
def test_far_offsets(device):
    """Elements beyond 2^32 of a tensor (rows of a 9 GiB buffer, the last ones looked at)."""
    from qmoe import block_norm, token_logprobs
    V, T = 131072, 36000
    buf = torch.empty((T, V), dtype=BF16, device=device)
    buf.zero_()
    g = gen(device, 6)
    buf[T - 3:] = rows(g, 3, V, BF16)
    tok = torch.full((T,), 17, device=device, dtype=torch.int64)
    log("far logits")
    got = token_logprobs(buf, tok, top=3)
    want = R.token_logprobs(buf[T - 3:], tok[T - 3:], 3)
    R.assert_close(got.logprobs[T - 3:], *want[0], "logprobs")
    R.assert_close(got.entropy[T - 3:], *want[1], "entropy")
    assert torch.equal(got.top_ids[T - 3:], want[2]) and got.top_ids[:T - 3].eq(torch.arange(3, device=device)).all()
    log("far rows")
    x = buf.view(-1, 2048)
    w = torch.ones(2048, dtype=BF16, device=device)
    out = block_norm(x, w)
    R.assert_close(out[-100:], *R.block_norm(x[-100:], w), "block_norm")
    assert out[:1000].eq(0).all()


@pytest.mark.gpu
def test_graphs_and_streams(device):
    """Captured and replayed with new inputs, eager work between the replays; two graphs and two
    streams at once."""
    from qmoe import block_residual, token_logprobs
    g = gen(device, 8)
    T, V, H = 3, 50003, 2560
    w = torch.ones(H, dtype=BF16, device=device)

    def step(s):
        h, x = block_residual(s["y"], s["r"], post_weight=w, gate=s["g"], gate_act="sigmoid", next_weight=w)
        return (h, x, *token_logprobs(s["l"], s["t"], top=7))

    def fill(s):
        s["y"].copy_(torch.randn((T, H), generator=g, device=device))
        s["r"].copy_(torch.randn((T, H), generator=g, device=device))
        s["g"].copy_(torch.randn((T, 1), generator=g, device=device))
        s["l"].copy_(rows(g, T, V, BF16))
        s["t"].copy_(torch.randint(0, V, (T,), generator=g, device=device))

    def state():
        s = dict(y=torch.empty((T, H), dtype=BF16, device=device), r=torch.empty((T, H), dtype=BF16, device=device),
                 g=torch.empty((T, 1), dtype=BF16, device=device), l=torch.empty((T, V), dtype=BF16, device=device),
                 t=torch.empty((T,), dtype=torch.int64, device=device))
        fill(s)
        return s

    states, graphs, outs = [state(), state()], [], []
    for s in states:
        log("capture")
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(s))
        graphs.append(gr)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(4):
        log(f"replay {rep}")
        for s in states:
            fill(s)
        torch.cuda.synchronize()
        eager = [tuple(t.clone() for t in step(s)) for s in states]
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for out, want in zip(outs, eager):
            assert all(torch.equal(a, b) for a, b in zip(out, want))
        res = []
        for s, st in zip(states, streams):
            with torch.cuda.stream(st):
                res.append([step(s) for _ in range(3)])
        torch.cuda.synchronize()
        for rs, want in zip(res, eager):
            for r in rs:
                assert all(torch.equal(a, b) for a, b in zip(r, want))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 4, 37])
def test_layer_to_logprobs(device, T):
    """As a model runs them: the norm, the MoE block, its residual sum with the final norm, the W8
    lm_head, the tokens' scores; each operator checked on what it was given."""
    from gpu_util import layer, layer_dev
    from qmoe import DenseW8, block_norm, block_residual, token_logprobs
    from qmoe.shared import moe_block
    H, MI, E, k, V = 512, 128, 64, 8, 4000
    log(f"layer to logprobs T={T}")
    g = gen(device, T)
    gu, dn = layer_dev(layer(E, H, MI, 64, 3), device)
    rand = lambda *s, std=1.0: (torch.randn(s, generator=g, device=device) * std).to(BF16)
    sh_gu, sh_dn = rand(2 * MI + 1 + E, H, std=0.04), rand(H, MI, std=0.05)
    w1, wp, w2 = (rand(H, std=0.1) for _ in range(3))
    head = DenseW8(torch.randint(-127, 128, (V, H), generator=g, device=device, dtype=torch.int8),
                   rand(V, H // 128, std=0.0005).abs())
    h0 = rand(T, H, std=2.0)
    x = block_norm(h0, w1, offset=1.0)
    y = moe_block(x, sh_gu, sh_dn, gu, dn, k)
    kw = dict(post_weight=wp, next_weight=w2, scale=0.7, offset=1.0)
    h, xf = block_residual(y, h0, **kw)
    logits = head(xf)
    tok = torch.randint(0, V, (T,), generator=g, device=device)
    got = token_logprobs(logits, tok, top=5)
    R.assert_close(x, *R.block_norm(h0, w1, offset=1.0), "x")
    for a, e, name in zip((h, xf), R.block_residual(y, h0, **kw), ("h", "xf")):
        R.assert_close(a, *e, name)
    want = R.token_logprobs(logits, tok, 5)
    R.assert_close(got.logprobs, *want[0], "logprobs")
    R.assert_close(got.entropy, *want[1], "entropy")
    assert torch.equal(got.top_ids, want[2])


@pytest.mark.gpu
def test_logprobs_with_gradients(device):
    from qmoe import token_logprobs
    x = torch.zeros((2, 8), device=device, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward pass"):
        token_logprobs(x)
    with torch.no_grad():
        assert token_logprobs(x).entropy.shape == (2,)


@pytest.mark.gpu
def test_forward_mode(device):
    """Operands with a forward-mode tangent are refused; their primal values are taken."""
    from torch.autograd import forward_ad
    from qmoe import block_norm, block_residual, token_logprobs
    x, w = torch.ones((2, 8), device=device), torch.ones(8, device=device)
    want = block_norm(x, w), block_residual(x, x, next_weight=w)[1], token_logprobs(x).entropy
    with forward_ad.dual_level():
        d, dw = forward_ad.make_dual(x, x), forward_ad.make_dual(w, w)
        for call in (lambda: block_norm(d, w), lambda: block_norm(x, dw), lambda: block_residual(x, d),
                     lambda: block_residual(x, x, gate=d), lambda: token_logprobs(d)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        p = forward_ad.unpack_dual(d).primal
        got = block_norm(p, w), block_residual(p, p, next_weight=w)[1], token_logprobs(p).entropy
    assert all(torch.equal(a, b) for a, b in zip(got, want))
