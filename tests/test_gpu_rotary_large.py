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


T = (1 << 26) + 5  # tokens of one head of 8, 64 threads each: past 2^32 in all
STEP = 1 << 24


def tokens(device, seed):
    n = normal(device, seed)
    return torch.cat([n(min(STEP, T - at), 1, 8) for at in range(0, T, STEP)])


def test_rotate_past_a_row_of_the_grid(device):
    from qmoe import Rotary, rotate
    log(f"rotate T={T}")
    x, p = tokens(device, 1), torch.arange(T, dtype=torch.int32, device=device)
    for layout in ("half", "interleaved"):
        r = Rotary(8, layout=layout, device=device)
        out = rotate(x, p, r)
        for at in range(0, T, STEP):
            assert torch.equal(out[at:at + STEP], rotate(x[at:at + STEP], p[at:at + STEP], r)), at
    assert rotate(x, p, r, inplace=True) is x and torch.equal(x, out)


def test_append_past_a_row_of_the_grid(device):
    from qmoe import Rotary, append_kv, rotate
    log(f"append T={T}")
    page = 4096
    pages = -(-T // page)
    k, v = tokens(device, 2), tokens(device, 3)
    k_cache, v_cache = (torch.zeros((pages, page, 1, 8), dtype=torch.bfloat16, device=device) for _ in range(2))
    table = torch.arange(pages, dtype=torch.int32, device=device)[None]
    lengths = torch.tensor([T], dtype=torch.int32, device=device)
    starts = torch.tensor([0, T], dtype=torch.int32, device=device)
    r = Rotary(8, device=device)
    q = append_kv(k, v, k_cache, v_cache, table, lengths, starts=starts, rotary=r, q=k)
    p = torch.arange(T, dtype=torch.int32, device=device)
    for at in range(0, T, STEP):
        assert torch.equal(q[at:at + STEP], rotate(k[at:at + STEP], p[at:at + STEP], r)), at
    assert torch.equal(k_cache.flatten(0, 1)[:T], q) and torch.equal(v_cache.flatten(0, 1)[:T], v)
    assert not k_cache.flatten(0, 1)[T:].any()
