"""paged_attention at head sizes and lengths where its ways to cut the work meet: tiles in pieces and rows in many
parts for heads that do not fill their rows in LDS, many rows of one key head over long contexts, wide
tables, batches against the rules."""
import pytest
import torch

import attention_ref as A
from operators_ref import assert_close
from test_gpu_attention import check
from test_gpu_rotary import batch, log, normal

BF16, F16 = torch.bfloat16, torch.float16
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [72, 80, 96, 104, 112, 120, 136, 192, 248])
@pytest.mark.parametrize("new,before,window,dtype", [(300, 9000, 0, BF16), (300, 9000, 5000, F16), (40, 20000, 0, F16)])
def test_pieces(device, D, new, before, window, dtype):
    """Tiles of 128 rows whose keys are cut into pieces."""
    check(device, [new], [new + before], 16, 6, 2, D, dtype, window, seed=D)


@pytest.mark.parametrize("D", [80, 96, 112, 128, 192, 256])
@pytest.mark.parametrize("lengths", [[99000], [60000, 1, 45000]])
def test_many_parts(device, D, lengths):
    """One key head's keys over nearly all workgroups."""
    check(device, [1] * len(lengths), lengths, 64, 8, 1, D, BF16, seed=D)


@pytest.mark.parametrize("new,lengths,Hq,Hkv,D", [([1], [131072], 64, 1, 128), ([1, 1], [70000, 33000], 40, 1, 192), ([1] * 5, [50000, 3, 0, 1600, 9000], 64, 1, 64),
                                                  ([5], [131072], 8, 1, 128), ([5, 1, 9], [90000, 40000, 3000], 16, 2, 256),
                                                  ([17, 2], [66000, 30000], 40, 1, 96)])
def test_many_rows_over_long_contexts(device, new, lengths, Hq, Hkv, D):
    """33 to 128 rows of a key head, and more, each on all keys."""
    check(device, new, lengths, 16, Hq, Hkv, D, BF16, seed=D)
    check(device, new, lengths, 64, Hq, Hkv, D, F16, window=20000, seed=D + 1)


@pytest.mark.parametrize("D", [104, 112, 120])
@pytest.mark.parametrize("dtype,window", [(BF16, 0), (F16, 50)])
def test_heads_of_104_to_120(device, D, dtype, window):
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 0, 127, 128, 129, 300, 1000]
    check(device, [1] * len(lengths), lengths, 16, 8, 2, D, dtype, window, seed=D)
    check(device, [3, 0, 8, 1, 5, 2, 6], [3, 0, 200, 64, 1000, 66, 4], 16, 6, 3, D, dtype, window, seed=D, padding=3)
    check(device, [97, 0, 1, 300, 64], [97, 10, 777, 500, 63], 24, 8, 2, D, dtype, window, seed=D, padding=5)


@pytest.mark.parametrize("new,lengths", [([512], [512]), ([1024], [1024]), ([2048], [2048]), ([70, 1, 300], [70, 900, 1500]), ([1, 1], [4097, 3])])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (4, 1, 192)])
def test_wide_tables(device, new, lengths, Hq, Hkv, D):
    """Tables of 131072 tokens: the same sums, cut in another way."""
    from qmoe import paged_attention
    log(f"wide table new={new} {Hq}/{Hkv}x{D}")
    caches, table, lens, starts = batch(device, 4, new, lengths, 16, Hkv, D, BF16)
    wide = torch.full((len(new), 131072 // 16), -1, dtype=torch.int32, device=device)
    wide[:, :table.shape[1]] = table
    q = normal(device, 5)(sum(new), Hq, D, std=2.0)
    given = None if max(new) == 1 else starts
    want = A.attention(q, *caches, table, lens, starts)
    for t in (table, wide):
        assert_close(paged_attention(q, *caches, t, lens, starts=given), *want, "attention")


@pytest.mark.parametrize("times,tokens,before,window", [(2, 300, 3000, 0), (2500, 4096, 61440, 0), (2500, 4096, 61440, 9000), (70, 5, 30000, 0)])
def test_starts_against_the_rules_write_nothing_else(device, times, tokens, before, window):
    """Sequences that share rows, once with more keys in all than 32 bits count: nothing is written before or behind the
    output and the workspace."""
    from qmoe import _lib
    L = _lib.lib()
    log(f"starts out of order: {times} x {tokens} window={window}")
    Hq, Hkv, D, page, pad = 32, 8, 64, 64, 1 << 20
    n = normal(device, 5)
    caches = [n(2, page, Hkv, D, dtype=F16) for _ in range(2)]
    B = 2 * times - 1
    table = torch.zeros((B, -(-(tokens + before) // page)), dtype=torch.int32, device=device)
    lens = torch.full((B,), tokens + before, dtype=torch.int32, device=device)
    starts = torch.tensor([0, tokens] * times, dtype=torch.int32, device=device)
    q = n(tokens, Hq, D, dtype=F16)
    need = L.qmoe_paged_attention_workspace(tokens, B, Hq, Hkv, D, page, table.shape[1], 0)
    assert need > 0
    ws, out = (torch.full((size + 2 * pad,), 171, dtype=torch.uint8, device=device) for size in (need, 2 * q.numel()))
    rc = L.qmoe_paged_attention(
        q.data_ptr(), q.stride(0), q.stride(1), caches[0].data_ptr(), *caches[0].stride()[:3], caches[1].data_ptr(),
        *caches[1].stride()[:3], 1, table.data_ptr(), table.stride(0), table.shape[1], lens.data_ptr(), starts.data_ptr(),
        out.data_ptr() + pad, tokens, B, Hq, Hkv, D, page, caches[0].shape[0], 0.125, window, ws.data_ptr() + pad, need, _lib.stream_of(q))
    assert rc == 0
    for t in (ws, out):
        assert (t[:pad] == 171).all() and (t[-pad:] == 171).all()
