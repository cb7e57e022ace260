"""What the norm and log-probability operators refuse, and their references (CPU only)."""
import math

import pytest
import torch

import operators_ref as R

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def t(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("call,says", [
    (lambda q: q.block_norm(t(2, 8), t(8)), "device tensors"),
    (lambda q: q.block_norm(t(2, 8), t(7)), "weight"),
    (lambda q: q.block_norm(t(2, 8), t(8, dtype=torch.float64)), "weight"),
    (lambda q: q.block_norm(t(2, 8, dtype=torch.int32), t(8)), "x must be"),
    (lambda q: q.block_norm(t(2, 0), t(0)), "1 <= H"),
    (lambda q: q.block_norm(t(2, 32769), t(32769)), "1 <= H"),
    (lambda q: q.block_norm(torch.zeros((), dtype=BF16), t(1)), "1 <= H"),
    (lambda q: q.block_norm(t(2, 8), t(8), out_dtype=F32), "out_dtype"),
    (lambda q: q.block_norm(t(2, 8), t(8), out_dtype=F16), "out_dtype"),
    (lambda q: q.block_residual(t(2, 8), t(2, 8)), "device tensors"),
    (lambda q: q.block_residual(t(2, 8), t(8)), "do not match"),
    (lambda q: q.block_residual(t(2, 8), t(2, 8, dtype=F16)), "residual must have"),
    (lambda q: q.block_residual(t(2, 8, dtype=F32), t(2, 8)), "residual must have"),
    (lambda q: q.block_residual(t(2, 8), t(2, 8), gate=t(2, 1), gate_act="tanh"), "gate_act"),
    (lambda q: q.block_residual(t(2, 8), t(2, 8), gate_act="sigmoid"), "needs a gate"),
    (lambda q: q.block_residual(t(2, 8), t(2, 8), gate=t(2, 1, dtype=torch.int8)), "gate must be"),
    (lambda q: q.block_residual(t(2, 8), t(2, 8), post_weight=t(2, 8)), "post_weight"),
    (lambda q: q.block_residual(t(2, 8), t(2, 8), next_weight=t(9)), "next_weight"),
    (lambda q: q.token_logprobs(t(2, 8)), "device tensors"),
    (lambda q: q.token_logprobs(t(2, 8, dtype=torch.int64)), "logits must be"),
    (lambda q: q.token_logprobs(t(2, 0)), "1 <= V"),
    (lambda q: q.token_logprobs(t(2, 8), top=33), "top"),
    (lambda q: q.token_logprobs(t(2, 8), top=-1), "top"),
    (lambda q: q.token_logprobs(t(2, 8), torch.zeros(2, dtype=torch.int32)), "int64"),
    (lambda q: q.token_logprobs(t(2, 8), torch.zeros(3, dtype=torch.int64)), "do not match"),
    (lambda q: q.token_logprobs(t(2, 8), torch.zeros((2, 3, 1), dtype=torch.int64)), "do not match"),
    (lambda q: q.token_logprobs(t(2, 8), allowed=torch.ones((2, 7), dtype=torch.bool)), "allowed"),
    (lambda q: q.token_logprobs(t(2, 8), allowed=torch.ones((2, 8), dtype=torch.uint8)), "allowed"),
])
def test_refusals(call, says):
    import qmoe
    with pytest.raises(RuntimeError, match=says):
        call(qmoe)


def test_gate_that_does_not_broadcast():
    from qmoe.norms import _gate_steps
    with pytest.raises(RuntimeError, match="does not broadcast"):
        _gate_steps(t(3, 1), (2, 8), 8)
    assert _gate_steps(t(2, 1), (2, 8), 8)[1:] == (1, 0)
    assert _gate_steps(t(8), (2, 8), 8)[1:] == (0, 1)
    assert _gate_steps(t(1, 1), (2, 8), 8)[2] == 0
    assert _gate_steps(t(2, 3, 1), (2, 3, 8), 8)[1:] == (1, 0)
    assert _gate_steps(t(8, 2).t(), (2, 8), 8)[1:] == (8, 1)     # columns first: copied
    assert _gate_steps(t(2, 16)[:, :8], (2, 8), 8)[1:] == (16, 1)


def test_inplace_overlap():
    from qmoe.norms import _inplace_rows
    base = t(64)
    r = base[:32].view(4, 8)
    assert _inplace_rows(r, 8, ((r, True), (None, False))).data_ptr() == r.data_ptr()
    for other, fine in ((r, False), (base[8:40].view(4, 8), True), (base[31:39], False)):
        with pytest.raises(RuntimeError, match="overlaps"):
            _inplace_rows(r, 8, ((other, fine),))
    _inplace_rows(r, 8, ((base[32:].view(4, 8), False),))
    wide = t(4, 20)                       # columns of the same rows, beside each other or not
    r = wide[:, 2:10]
    for cols, fine in ((slice(10, 18), True), (slice(12, 20), True), (slice(9, 17), False), (slice(0, 2), True),
                       (slice(1, 3), False), (slice(18, 20), True)):
        if fine:
            _inplace_rows(r, 8, ((wide[:, cols], False),))
        else:
            with pytest.raises(RuntimeError, match="overlaps"):
                _inplace_rows(r, 8, ((wide[:, cols], True),))
    _inplace_rows(r, 8, ((wide[:, 19:].expand(4, 8), False),))      # one gate per row, beside the rows
    with pytest.raises(RuntimeError, match="overlaps"):
        _inplace_rows(r, 8, ((wide[:, 9:10].expand(4, 8), False),))
    with pytest.raises(RuntimeError, match="overlaps"):             # wraps into the next row
        _inplace_rows(r, 8, ((wide.view(-1)[18:18 + 60].view(3, 20)[:, :6], False),))
    one = base.as_strided((1, 8), (0, 1))  # a single row may have any step
    _inplace_rows(one, 8, ((base.as_strided((1, 8), (0, 1), 8), False), (one, True)))
    with pytest.raises(RuntimeError, match="overlaps"):
        _inplace_rows(one, 8, ((base.as_strided((1, 8), (0, 1), 4), True),))
    with pytest.raises(RuntimeError, match="do not overlap"):
        _inplace_rows(t(1, 8).expand(4, 8), 8, ())
    with pytest.raises(RuntimeError, match="do not overlap"):
        _inplace_rows(base[:32].view(8, 4).t(), 8, ())


class Operand:
    def __init__(self, device=0, requires_grad=False):
        self.device_index, self.requires_grad = device, requires_grad

    def get_device(self):
        return self.device_index


def test_operands(monkeypatch):
    """Gradients, host tensors and two devices are refused; another device than the current one is
    told apart."""
    from qmoe import _lib
    monkeypatch.setattr(_lib, "current_device", lambda: 0)
    assert _lib.operands(Operand(), None, Operand()) is True
    assert _lib.operands(Operand(1), Operand(1)) is False
    for ops, says in (([Operand(-1)], "device tensors"), ([Operand(), Operand(-1)], "device tensors"),
                      ([Operand(-1), Operand()], "device tensors"), ([Operand(), None, Operand(1)], "same device"),
                      ([Operand(requires_grad=True)], "no backward pass"),
                      ([Operand(), Operand(requires_grad=True)], "no backward pass")):
        with pytest.raises(RuntimeError, match=says):
            _lib.operands(*ops)
    with torch.no_grad():
        assert _lib.operands(Operand(requires_grad=True), Operand(requires_grad=True))


def test_c_entries_refuse_before_any_launch():
    from qmoe import _lib
    L = _lib.lib()

    def norm(rows=1, H=8, eps=1e-6, offset=0.0, xt=0, wt=0, yt=0, ldx=8, ldy=8, p=None):
        return L.qmoe_block_norm(p, ldx, xt, p, wt, p, ldy, yt, rows, H, eps, offset, None)
    assert norm(rows=0) == 0
    for kw in (dict(rows=-1), dict(H=0), dict(H=32769, ldy=32769), dict(eps=0.0), dict(eps=-1.0), dict(eps=1e-31),
               dict(eps=math.nan), dict(eps=math.inf), dict(offset=math.nan), dict(wt=3), dict(ldx=-1), dict(ldy=7)):
        assert norm(**kw) == -1 and norm(**{"rows": 0, **kw}) == -1, kw
    assert norm() == -1  # null pointers

    def res(rows=1, H=8, yt=0, rt=0, gate=None, g_row=1, g_col=0, gt=0, scale=1.0, h=None, ldr=8, ldh=8, nxt=None,
            x=None, ldx=8, r=None, y=None):
        return L.qmoe_block_residual(y, 8, yt, r, ldr, rt, None, 0, gate, g_row, g_col, gt, 0, scale, h, ldh, nxt, 0,
                                     x, ldx, rows, H, 1e-6, 0.0, None)
    assert res(rows=0) == 0
    for kw in (dict(rows=-1), dict(scale=math.inf), dict(gate=16, gt=7), dict(gate=16, g_col=2), dict(gate=16, g_row=-1),
               dict(nxt=16), dict(x=16), dict(nxt=16, x=16, ldx=7), dict(ldr=-1), dict(ldh=7)):
        assert res(**{"rows": 0, **kw}) == -1, kw
    assert res() == -1
    assert res(y=16, r=32, h=32, ldr=16, ldh=8) == -1       # in place with another row step
    assert res(y=16, r=32, h=48, yt=0, rt=1) == -1          # types that do not go together
    assert res(y=16, r=32, h=48, yt=2, rt=0) == -1

    def lp(T=1, V=8, kind=0, m=0, top=0, ld=8, p=None, allowed=None, lda=0):
        return L.qmoe_token_logprobs(p, ld, kind, p, m, allowed, lda, T, V, p, p, top, p, p, None, 0, None)
    assert lp(T=0) == 0
    for kw in (dict(T=-1), dict(V=0), dict(V=(1 << 30) + 1), dict(m=-1), dict(top=33), dict(top=-1), dict(ld=-1),
               dict(allowed=16, lda=-1)):
        assert lp(**kw) == -1, kw
    assert lp() == -1


@pytest.mark.parametrize("T,V,kind,parts", [
    (1, 131072, 0, 64), (1, 32768, 0, 1), (1, 32776, 0, 17), (1, 1 << 30, 0, 64), (16, 131072, 0, 64), (48, 131072, 0, 16),
    (64, 65536, 0, 1), (63, 65536, 0, 16), (64, 131072, 0, 16), (100, 131072, 1, 8), (127, 131072, 1, 8),
    (128, 131072, 1, 1), (159, 262144, 0, 6), (160, 1 << 30, 2, 1), (512, 1 << 30, 2, 1), (1, 16384, 2, 1),
    (1, 16388, 2, 17), (3, 7, 0, 1), (2, 1000003, 0, 62),
])
def test_parts_of_rows(T, V, kind, parts):
    """How token_logprobs splits rows over workgroups, by its workspace: 12 bytes of sums and 8 bytes per
    candidate for each part."""
    from qmoe import _lib
    ws = _lib.lib().qmoe_token_logprobs_workspace
    n = T * parts
    assert ws(T, V, kind, 0) == (0 if parts == 1 else -(-12 * n // 16) * 16)
    assert ws(T, V, kind, 20) - ws(T, V, kind, 0) == (0 if parts == 1 else 160 * n)


def test_references():
    """The references against hand-worked values and torch's own float64 functions."""
    out, err = R.block_norm(torch.tensor([[3.0, 4.0]]), torch.tensor([1.0, 2.0]), eps=12.5)
    assert torch.allclose(out, torch.tensor([[0.6, 1.6]], dtype=torch.float64)) and (err < 1e-5).all()
    (h, _), (x, _) = R.block_residual(torch.tensor([[2.0, 0.0]]), torch.tensor([[1.0, 4.0]]), scale=0.5,
                                      gate=torch.tensor([[4.0]]), next_weight=torch.tensor([1.0, 1.0]), eps=1e-9)
    assert h.tolist() == [[5.0, 4.0]] and torch.allclose(x, h / math.sqrt(20.5))
    g = torch.Generator().manual_seed(0)
    l = torch.randn((3, 50), generator=g) * 3
    l[1, 7:] = -float("inf")
    tok = torch.tensor([[1, -1], [9, 50], [4, 4]])
    (lp, _), (ent, _), ids, (tl, _) = R.token_logprobs(l, tok, top=8)
    ref = l.double().log_softmax(1)
    assert torch.allclose(lp[0, 0], ref[0, 1]) and lp[0, 1] == 0 and lp[1, 0] == -math.inf and lp[1, 1].isnan()
    want = torch.distributions.Categorical(logits=l.double()[[0, 2]]).entropy()
    assert torch.allclose(ent[[0, 2]], want)
    assert ids[0].tolist() == torch.topk(l[0], 8)[1].tolist() and ids[1, 7] == -1 and tl[1, 7] == -math.inf
    (_, _), (ent, _), ids, _ = R.token_logprobs(torch.tensor([[math.nan, 1.0], [-math.inf, -math.inf]]),
                                                torch.tensor([0, 0]), top=1)
    assert ent[0].isnan() and ent[1] == 0 and ids.tolist() == [[-1], [-1]]


def test_planted_mistakes_are_seen():
    """assert_close tells an exact value from one a step of the type away, and other infinities and NaN."""
    e = torch.tensor([1.0, 100.0, 0.0, math.nan, -math.inf], dtype=torch.float64)
    b = R.half_step(e, BF16)
    R.assert_close(e.to(BF16), e, b, "same")
    for at, v in ((0, 1.0 + 2 ** -7), (1, 100.5), (2, 1e-30), (3, 0.0), (4, math.inf), (0, math.nan)):
        g = e.clone()
        g[at] = v
        with pytest.raises(AssertionError):
            R.assert_close(g.to(BF16), e, b, "planted")


def negated(*shape, dtype=torch.complex64):
    """A view with the values -1, -2, ... and the memory 1, 2, ... (a step of 2 apart)."""
    n = math.prod(shape)
    z = torch.complex(*(torch.arange(1.0, n + 1).view(shape).to(F16 if dtype == torch.complex32 else F32),) * 2)
    return torch.imag(z.conj())


@pytest.mark.parametrize("dtype", [torch.complex64, torch.complex32])
def test_negated_views(dtype):
    """Operands whose memory holds the other sign are handed on with their values in memory."""
    from qmoe.norms import _check_weight, _gate_steps, _inplace_rows, _rows
    v = negated(4, 1, dtype=dtype)
    assert v.is_neg()
    want = [-1.0, -2.0, -3.0, -4.0]
    for got in (_rows(v, 1), _rows(v.view(2, 2, 1), 1), _gate_steps(v, (4, 8), 8)[0],
                _gate_steps(v, (4, 1), 1)[0], _gate_steps(v.view(2, 2, 1), (2, 2, 8), 8)[0][:, :1]):
        assert not got.is_neg() and got.flatten().tolist() == want
    for got in (_check_weight(v[:1, 0], 1, "weight"), _check_weight(v[:, 0], 4, "weight")):
        assert not got.is_neg() and got.tolist() == want[:got.numel()]
    plain = torch.ones(3, 4)
    assert _rows(plain, 4) is plain
    with pytest.raises(RuntimeError, match="negated"):
        _inplace_rows(v, 1, ())


def test_forward_mode_tangents_are_refused(monkeypatch):
    """A dual tensor does not require a gradient, and its tangent would be lost."""
    from torch.autograd import forward_ad
    from qmoe import _lib
    monkeypatch.setattr(_lib, "current_device", lambda: 0)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    x = torch.ones(2, 8)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        assert not dual.requires_grad
        for ops in ((dual,), (x, None, dual)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                _lib.operands(*ops)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                _lib.operands(*ops)
        assert _lib.operands(x, None, forward_ad.unpack_dual(dual).primal) is True
        with monkeypatch.context() as m:  # without the name that tells whether a level is entered
            m.delattr(forward_ad, "_current_level")
            m.setattr(forward_ad, "unpack_dual", lambda t, f=forward_ad.unpack_dual: f(t, level=0))
            assert _lib.operands(x) is True
            with pytest.raises(RuntimeError, match="forward-mode"):
                _lib.operands(dual)
    assert _lib.operands(x, dual) is True


def test_many_tokens_per_row():
    """More than 2^30 tokens for a row are refused: the kernels count them in 32 bits, a workgroup's
    stride on top (checked before anything is read; the pointers are not real)."""
    import qmoe
    from qmoe import _lib
    L = _lib.lib()
    for m in ((1 << 30) + 1, (1 << 31) - 256, (1 << 31) - 1):
        for T in (0, 1):
            assert L.qmoe_token_logprobs(16, 8, 0, 16, m, None, 0, T, 8, 16, 16, 0, None, None, None, 0, None) == -1, m
    assert L.qmoe_token_logprobs(16, 8, 0, 16, 1 << 30, None, 0, 0, 8, 16, 16, 0, None, None, None, 0, None) == 0
    one = torch.zeros((), dtype=torch.int64)
    for m in ((1 << 30) + 1, 1 << 31, (1 << 32) + 5):
        with pytest.raises(RuntimeError, match="2.30 for each row"):
            qmoe.token_logprobs(t(2, 8), one.expand(2, m))
    with pytest.raises(RuntimeError, match="device tensors"):
        qmoe.token_logprobs(t(2, 8), one.expand(2, 1 << 30))


def test_gates_of_a_batch():
    """One value per sequence stays one value per row; only as many values as rows are ever copied."""
    from qmoe.norms import _gate_steps
    for shape, of, want in (((2, 1, 1), (2, 5, 8), [0] * 5 + [1] * 5), ((1, 5, 1), (2, 5, 8), [0, 1, 2, 3, 4] * 2),
                            ((5, 1), (2, 5, 8), [0, 1, 2, 3, 4] * 2), ((), (2, 5, 8), [0] * 10), ((1,), (8,), [0]),
                            ((2, 1, 2, 1), (2, 3, 2, 8), [0, 1] * 3 + [2, 3] * 3), ((2, 5, 1), (2, 5, 1), list(range(10))),
                            ((2, 1, 1), (2, 0, 8), [])):
        gate = torch.arange(float(math.prod(shape))).view(shape)
        g, row, column = _gate_steps(gate, of, of[-1])
        assert column == 0 and g.untyped_storage().nbytes() <= 4 * max(gate.numel(), len(want)), shape
        assert g.as_strided((len(want),), (row,)).tolist() == want, shape


def test_workspace_is_checked_before_any_launch():
    """Split rows need their workspace: none, one that is too short or off its alignment is refused (no
    pointer here is real). The need does not grow with the rows: a size is good for its own call only."""
    from qmoe import _lib
    L = _lib.lib()
    size = L.qmoe_token_logprobs_workspace
    EWORKSPACE = -2

    def call(T, V, top, ws, nbytes, kind=0):
        return L.qmoe_token_logprobs(16, V, kind, 16, 1, None, 0, T, V, 16, 16, top, 16, 16, ws, nbytes, None)
    for T, V, top, kind in ((1, 131072, 20, 0), (1, 131072, 0, 0), (48, 131072, 8, 1), (127, 131072, 32, 0), (159, 262144, 5, 0),
                            (1, 16388, 1, 2), (3, 1 << 30, 20, 0)):
        need = size(T, V, kind, top)
        assert need > 0 and need % 8 == 0
        for ws, nbytes in ((None, need), (None, 0), (4096, need - 1), (4096, 0), (4096 + 8, need), (4096 + 1, need + 64)):
            assert call(T, V, top, ws, nbytes, kind) == EWORKSPACE, (T, V, top, ws, nbytes)
    assert size(127, 131072, 0, 20) > size(128, 131072, 0, 20) == 0
    assert size(16, 131072, 0, 20) > size(17, 131072, 0, 20) and size(1, 131072, 0, 20) > size(1, 131080, 0, 20)
    assert call(127, 131072, 20, 4096, size(128, 131072, 0, 20)) == EWORKSPACE
    assert call(127, 131072, 20, 4096, size(127, 131072, 0, 8)) == EWORKSPACE
