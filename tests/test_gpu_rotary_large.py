"""rotate and append_kv on many tokens."""
import pytest
import torch

from test_gpu_rotary import batch, log, normal

BF16, F32 = torch.bfloat16, torch.float32
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,D,rd", [((32, 8), 128, 128), ((8, 2), 80, 40), ((16, 2), 256, 64)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_bits_do_not_depend_on_the_call(device, heads, D, rd, dtype, layout):
    """A long prompt stored and turned at once and in chunks, down to single tokens: the same bits."""
    from qmoe import Rotary, append_kv, rotate
    log(f"long prompt {heads} x {D} {dtype} {layout}")
    Hq, Hkv = heads
    T = 12000
    n = normal(device, D)
    q, k, v = n(T, Hq, D, dtype=dtype), n(T, Hkv, D, dtype=dtype), n(T, Hkv, D, dtype=dtype)
    r = Rotary(rd, 1.0e6, layout=layout, device=device)
    results = []
    for steps in ([T], [11000, 600] + [1] * 8 + [392]):
        caches, table, _, _ = batch(device, 1, [T], [T], 16, Hkv, D, dtype)
        out, at = [], 0
        for step in steps:
            rows = slice(at, at + step)
            at += step
            lengths, starts = (torch.tensor(x, dtype=torch.int32, device=device) for x in ([at], [0, step]))
            out.append(append_kv(k[rows], v[rows], *caches, table, lengths, starts=starts, rotary=r, q=q[rows]))
        results.append((torch.cat(out), *caches))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    p = torch.arange(T, device=device)
    assert torch.equal(rotate(q, p, r), results[0][0])
    assert torch.equal(torch.cat([rotate(q[i:i + 7], p[i:i + 7], r) for i in range(0, 70, 7)]), results[0][0][:70])
