"""rotate, append_kv and paged_attention as a model uses them: one after the other over many steps, in captured graphs, on
streams side by side, under inference mode."""
import pytest
import torch

import attention_ref as A
from operators_ref import assert_close
from test_gpu_rotary import batch, log, normal

BF16, F16 = torch.bfloat16, torch.float16
pytestmark = pytest.mark.gpu


def layer(q, k, v, caches, table, lengths, starts, rotary, window=0):
    from qmoe import append_kv, paged_attention
    q = append_kv(k, v, *caches, table, lengths, starts=starts, rotary=rotary, q=q)
    return paged_attention(q, *caches, table, lengths, starts=starts, window=window)


@pytest.mark.parametrize("D,Hq,Hkv,window", [(128, 8, 2, 0), (64, 6, 6, 40), (256, 8, 1, 0)])
def test_prompt_in_steps(device, D, Hq, Hkv, window):
    """A prompt at once, in chunks and token by token: the same caches, outputs within the bounds of the formula."""
    from qmoe import Rotary, block_norm, block_residual, rotate
    log(f"prompt in steps D={D}")
    n, T = normal(device, D), 150
    H = Hq * D
    h, w = n(T, H, std=2.0), n(H, std=0.1)
    qkv = torch.randn((H, (Hq + 2 * Hkv) * D), device=device).div_(H ** 0.5).to(BF16)
    rotary = Rotary(D // 2, 1.0e4, layout="interleaved", device=device)
    x = block_norm(h, w, offset=1.0)
    heads = (x @ qkv).unflatten(1, (Hq + 2 * Hkv, D))
    q, k, v = heads.split((Hq, Hkv, Hkv), dim=1)
    results = []
    for steps in ([T], [100, 1, 49], [64, 64] + [1] * 22):
        caches, table, _, _ = batch(device, 1, [T], [T], 16, Hkv, D, BF16)
        out, at = [], 0
        for step in steps:
            lengths = torch.tensor([at + step], dtype=torch.int32, device=device)
            starts = torch.tensor([0, step], dtype=torch.int32, device=device)
            rows = slice(at, at + step)
            out.append(layer(q[rows], k[rows], v[rows], caches, table, lengths, starts if step > 1 else None, rotary, window))
            at += step
        results.append((caches, torch.cat(out)))
    turned = rotate(q, torch.arange(T, device=device), rotary)
    lengths, starts = torch.tensor([T]), torch.tensor([0, T])
    for caches, out in results:
        for a, b in zip(caches, results[0][0]):
            assert torch.equal(a, b)
        assert_close(out, *A.attention(turned, *caches, table, lengths, starts, None, window), "steps")
    y, _ = block_residual(results[0][1].flatten(1), h, next_weight=w, offset=1.0)
    assert y.isfinite().all()


@pytest.mark.parametrize("new", [[1] * 6, [1, 70, 3, 0, 200, 1], [5, 1, 2, 3, 4, 6]])
@pytest.mark.parametrize("D", [64, 256])
def test_graph(device, new, D):
    """A captured layer follows its lengths, tables and tokens; every replay gives the eager bits. A second graph,
    replayed on another stream at the same time, does not disturb it."""
    from qmoe import Rotary
    log(f"graph new={new} D={D}")
    Hq, Hkv, page, width = 8, 2, 16, 130
    rotary = Rotary(D, device=device)
    starts = None if max(new) == 1 else torch.tensor([sum(new[:b]) for b in range(7)], dtype=torch.int32, device=device)
    T = sum(new)

    def inputs(seed):
        g = torch.Generator(device=device).manual_seed(seed)
        cpu = torch.Generator().manual_seed(seed)
        lengths = torch.tensor([m + int(torch.randint(0, width * page - m, (1,), generator=cpu)) for m in new], dtype=torch.int32)
        qkv = torch.randn((T, Hq + 2 * Hkv, D), generator=g, device=device).to(BF16)
        table = torch.randperm(6 * width, generator=g, device=device).view(6, width).int()
        return qkv, lengths.to(device), table

    def make(stream):
        held = [t.clone() for t in inputs(0)]
        caches = [normal(device, 3)(6 * width, page, Hkv, D) for _ in range(2)]
        qkv, lengths, table = held
        run = lambda: layer(*qkv.split((Hq, Hkv, Hkv), 1), caches, table, lengths, starts, rotary)
        with torch.cuda.stream(stream):
            run()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = run()
        return held, caches, graph, out

    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs = [make(s) for s in streams]
    torch.cuda.synchronize()
    for seed in range(1, 5):
        fresh = [inputs(seed + 10 * i) for i in range(2)]
        before = []
        for (held, caches, _, out), new_inputs in zip(graphs, fresh):
            for t, f in zip(held, new_inputs):
                t.copy_(f)
            before.append([c.clone() for c in caches])
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        for stream, (_, _, graph, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, caches, _, out), kept, (qkv, lengths, table) in zip(graphs, before, fresh):
            eager = layer(*qkv.split((Hq, Hkv, Hkv), 1), kept, table, lengths, starts, rotary)
            assert torch.equal(out, eager)
            for a, b in zip(caches, kept):
                assert torch.equal(a, b)


def test_streams(device):
    """Calls on two streams at once, on tensors made on another, give what they give alone."""
    from qmoe import paged_attention
    log("two streams")
    sets = []
    for seed, new, lengths in ((1, [1] * 20, [3000 + 100 * b for b in range(20)]), (2, [400, 9], [2000, 5000])):
        caches, table, lens, starts = batch(device, seed, new, lengths, 16, 2, 128, F16)
        q = normal(device, seed)(sum(new), 16, 128, std=2.0, dtype=F16)
        sets.append((q, *caches, table, lens, starts))
    alone = [paged_attention(*s[:5], starts=s[5]) for s in sets]
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = [[], []]
    for _ in range(6):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(paged_attention(*sets[i][:5], starts=sets[i][5]))
    torch.cuda.synchronize()
    for want, outs in zip(alone, got):
        for out in outs:
            assert torch.equal(out, want)


def test_gradients_and_modes(device):
    """Leaves that require a gradient are refused while gradients are recorded, and taken under no_grad; inference
    tensors are written in place."""
    from qmoe import Rotary, append_kv, paged_attention, rotate
    caches, table, lens, starts = batch(device, 1, [3], [40], 16, 2, 64, BF16)
    q, k, v = (normal(device, i)(3, h, 64) for i, h in enumerate((4, 2, 2)))
    rotary, p = Rotary(64, device=device), torch.arange(3, device=device)
    want = layer(q, k, v, [c.clone() for c in caches], table, lens, starts, rotary)
    q.requires_grad_()
    for call in (lambda: rotate(q, p, rotary), lambda: append_kv(k, v, *caches, table, lens, starts=starts, q=q),
                 lambda: paged_attention(q, *caches, table, lens, starts=starts)):
        with pytest.raises(RuntimeError, match="no backward pass"):
            call()
    with torch.no_grad():
        assert torch.equal(layer(q, k, v, [c.clone() for c in caches], table, lens, starts, rotary), want)
    with torch.inference_mode():
        mine = [c.clone() for c in caches]
        assert torch.equal(layer(q, k, v, mine, table, lens, starts, rotary), want)
        x = k.clone()
        assert torch.equal(rotate(x, p, rotary, inplace=True), rotate(k, p, rotary))


def test_workspace(device):
    """The C entry takes a workspace of the size it names (and asks for one where keys are cut), and writes nothing
    behind it."""
    from qmoe import _lib, paged_attention
    L = _lib.lib()
    for new, lengths in (([1], [5000]), ([300], [9000]), ([1, 90, 4], [700, 3000, 64])):
        caches, table, lens, starts = batch(device, 1, new, lengths, 16, 2, 64, BF16)
        T, B, one = sum(new), len(new), int(max(new) == 1)
        q = normal(device, 2)(T, 8, 64)
        need = L.qmoe_paged_attention_workspace(T, B, 8, 2, 64, 16, table.shape[1], one)
        assert need > 0
        ws = torch.full((need + 4096,), 171, dtype=torch.uint8, device=device)
        out = torch.empty_like(q)
        log(f"workspace {need} new={new}")
        call = lambda n: L.qmoe_paged_attention(
            q.data_ptr(), q.stride(0), q.stride(1), caches[0].data_ptr(), *caches[0].stride()[:3], caches[1].data_ptr(),
            *caches[1].stride()[:3], 0, table.data_ptr(), table.stride(0), table.shape[1], lens.data_ptr(),
            None if one else starts.data_ptr(), out.data_ptr(), T, B, 8, 2, 64, 16, caches[0].shape[0], 0.125, 0,
            ws.data_ptr(), n, _lib.stream_of(q))
        assert call(need - 1) == -2 and call(0) == -2
        assert call(need) == 0
        assert torch.equal(out, paged_attention(q, *caches, table, lens, starts=None if one else starts))
        assert (ws[need:] == 171).all()


@pytest.mark.parametrize("times,tokens,before", [(2, 300, 3000), (2500, 4096, 61440)])
def test_starts_out_of_order(device, times, tokens, before):
    """Sequences that share rows against the rules, once with more keys in all than 32 bits count: results mean nothing
    then, but nothing is written outside of the output, and a call that keeps to the rules is right afterwards."""
    from qmoe import paged_attention
    log(f"starts out of order: {times} x {tokens}")
    Hq, Hkv, D, page = 32, 8, 64, 64
    n = normal(device, 5)
    caches = [n(2, page, Hkv, D, dtype=torch.float16) for _ in range(2)]
    B = 2 * times - 1
    table = torch.zeros((B, (tokens + before) // page), dtype=torch.int32, device=device)
    lens = torch.full((B,), tokens + before, dtype=torch.int32, device=device)
    starts = torch.tensor([0, tokens] * times, dtype=torch.int32, device=device)
    q = n(tokens, Hq, D, dtype=torch.float16)
    assert paged_attention(q, *caches, table, lens, starts=starts).shape == q.shape
    torch.cuda.synchronize()
    few = torch.tensor([0, 40], dtype=torch.int32, device=device)
    out = paged_attention(q[:40], *caches, table[:1], lens[:1], starts=few)
    assert_close(out, *A.attention(q[:40], *caches, table[:1], lens[:1], few), "attention")


@pytest.mark.parametrize("T,before,window", [(6000, 0, 4096), (3000, 0, 2000), (2600, 20000, 3000), (300, 9000, 0), (300, 9000, 5000),
                                             (2100, 3000, 0)])
def test_workspace_with_windows(device, T, before, window):
    """One sequence, tiles in pieces or whole: the workspace, which is asked for without the window, is enough."""
    from qmoe import paged_attention
    log(f"window {window}: {T} after {before}")
    caches, table, lens, starts = batch(device, 3, [T], [T + before], 16, 2, 64, BF16)
    q = normal(device, 4)(T, 20, 64, std=2.0, dtype=BF16)
    out = paged_attention(q, *caches, table, lens, starts=starts, window=window)
    assert_close(out, *A.attention(q, *caches, table, lens, starts, None, window), "attention")
