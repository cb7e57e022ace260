"""Timed cases of the operators of an attention layer over a paged cache.

* ``rotate``: rotary positions on the heads of each token;
* ``append``: the keys and values of new tokens written into the pages of their
  sequences, keys and queries rotated on the way;
* ``attend``: attention of the new tokens of a batch of sequences, one each or a chunk,
  over their pages.

Head layouts are generic ones (several query heads share a key and value head), head
sizes 64 to 256; batches go from one decoding sequence over many of different lengths to
prefill chunks. How many tokens a sequence has follows from the case alone (``mix`` seeds
it). All of it is called eagerly.

Inputs are made on the device from the seed: keys, values and new tokens N(0, 1), queries
N(0, 2) (scores of about N(0, 2) after the scale), pages in random order, a few spare ones
among them.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parent.parent / "qwen-ascend_amd")
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one decoding sequence: its query heads (the smallest call)
        {"name": "rotate_b1", "op": "rotate", "T": 1, "heads": 32, "D": 128, "rd": 128, "layout": "half", "x": "bf16",
         "scaling": "none", "factor": 1.0, "base": 1.0e6, "far": 32768, "pad": 0},
        # a long prefill: a quarter of each head turned, frequencies scaled by parts
        {"name": "rotate_t8192_part", "op": "rotate", "T": 8192, "heads": 16, "D": 256, "rd": 64, "layout": "half",
         "x": "bf16", "scaling": "parts", "factor": 4.0, "base": 1.0e6, "far": 131072, "pad": 0},
        # neighbouring elements as pairs, 32 bits, odd sizes, far positions, heads cut out of wider rows
        {"name": "rotate_odd_fp32", "op": "rotate", "T": 1003, "heads": 7, "D": 90, "rd": 54, "layout": "interleaved",
         "x": "fp32", "scaling": "linear", "factor": 8.0, "base": 1.0e4, "far": 4000000, "pad": 22},
        # a batch of decoding sequences: queries turned, keys turned and stored with the values
        {"name": "append_b64", "op": "append", "B": 64, "new": 1, "cached": 8192, "ragged": True, "mix": 11, "Hq": 32,
         "Hkv": 4, "D": 128, "rd": 128, "layout": "half", "page": 16, "x": "bf16"},
        # prefill chunks of three sequences
        {"name": "append_t4096", "op": "append", "B": 3, "new": 2048, "cached": 2048, "ragged": True, "mix": 12, "Hq": 32,
         "Hkv": 8, "D": 128, "rd": 128, "layout": "half", "page": 64, "x": "bf16"},
        # one decoding sequence
        {"name": "attend_b1", "op": "attend", "B": 1, "new": 1, "cached": 4096, "ragged": False, "mix": 1, "Hq": 32,
         "Hkv": 8, "D": 128, "page": 16, "x": "bf16", "window": 0},
        # a batch of decoding sequences of very different lengths
        {"name": "attend_b64_ragged", "op": "attend", "B": 64, "new": 1, "cached": 65536, "ragged": True, "mix": 2,
         "Hq": 32, "Hkv": 4, "D": 128, "page": 16, "x": "bf16", "window": 0},
        # a few long contexts with wide heads, two of them stored
        {"name": "attend_b4_long", "op": "attend", "B": 4, "new": 1, "cached": 131072, "ragged": False, "mix": 3,
         "Hq": 16, "Hkv": 2, "D": 256, "page": 64, "x": "bf16", "window": 0},
        # several proposed tokens for each sequence, checked at once; half precision
        {"name": "attend_b16_several", "op": "attend", "B": 16, "new": 5, "cached": 16384, "ragged": True, "mix": 4,
         "Hq": 24, "Hkv": 8, "D": 64, "page": 32, "x": "fp16", "window": 0},
        # a prompt from its start (the largest case)
        {"name": "attend_t8192", "op": "attend", "B": 1, "new": 8192, "cached": 0, "ragged": False, "mix": 5, "Hq": 32,
         "Hkv": 8, "D": 128, "page": 16, "x": "bf16", "window": 0},
        # chunks and single tokens in one batch, over what was cached before, wide heads
        {"name": "attend_mixed", "op": "attend", "B": 12, "new": 1024, "cached": 16384, "ragged": True, "mix": 6,
         "Hq": 16, "Hkv": 2, "D": 256, "page": 64, "x": "bf16", "window": 0},
        # a prompt under a sliding window, odd head size and group
        {"name": "attend_window", "op": "attend", "B": 2, "new": 6000, "cached": 3000, "ragged": True, "mix": 9, "Hq": 15,
         "Hkv": 3, "D": 80, "page": 16, "x": "fp16", "window": 1024},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rotate", "append", "attend", "attend", "attend", "attend"))
    mix = rng.randrange(1 << 30)
    if op == "rotate":
        x = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        D = rng.choice((64, 80, 96, 128, 192, 256, 2 * rng.randrange(4, 128)))
        rd = rng.choice((D, D, D // 2 // 2 * 2, 2 * rng.randrange(1, D // 2 + 1)))
        heads = _log_int(rng, 1, 64)
        scaling = rng.choice(("none", "none", "linear", "base", "parts")) if rd > 2 else "none"
        return {"op": op, "T": _log_int(rng, 1, max(1, min(16384, int(3.0e7 / (heads * D))))), "heads": heads, "D": D,
                "rd": rd, "layout": rng.choice(("half", "half", "interleaved")), "x": x, "scaling": scaling,
                "factor": 1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0)),
                "base": rng.choice((1.0e4, 5.0e5, 1.0e6)), "far": _log_int(rng, 1000, 4000000),
                "pad": rng.choice((0, 0, 16, 5))}
    Hkv, G = rng.choice((1, 2, 3, 4, 8)), rng.choice((1, 2, 3, 4, 5, 7, 8, 16))
    D = rng.choice((64, 80, 96, 128, 128, 192, 256))
    c = {"op": op, "Hq": Hkv * G, "Hkv": Hkv, "D": D, "page": rng.choice((16, 16, 32, 64, 128, 24)),
         "x": rng.choice(("bf16", "bf16", "fp16")), "ragged": rng.random() < 0.7, "mix": mix}
    kind = rng.choice(("single", "several", "chunk"))
    if op == "append":
        c["rd"] = rng.choice((D, D, D // 2))
        c["layout"] = rng.choice(("half", "half", "interleaved"))
        c["B"] = _log_int(rng, 1, 128 if kind == "single" else 16)
        c["new"] = {"single": 1, "several": rng.randrange(2, 9), "chunk": _log_int(rng, 16, 4096)}[kind]
        c["new"] = max(1, min(c["new"], int(2.5e7 / (c["B"] * (c["Hq"] + 2 * Hkv) * D))))
        c["cached"] = _log_int(rng, 1, max(1, int(2.0e7 / (c["B"] * Hkv * D))))
        return c
    c["window"] = 0 if rng.random() < 0.7 else _log_int(rng, 64, 4096)
    row = 2 * 2 * Hkv * D  # bytes of a cached token
    if kind == "chunk":
        c["B"] = _log_int(rng, 1, 8)
        most = int(2.0e11 / (4 * c["Hq"] * D * c["B"]))  # pairs of a new and a cached token, for each sequence
        c["new"] = _log_int(rng, 16, max(16, min(4096, int(math.sqrt(most)))))
        c["cached"] = _log_int(rng, 1, max(1, min(65536, most // c["new"])))
    else:
        c["B"] = _log_int(rng, 1, 128)
        c["new"] = 1 if kind == "single" else rng.randrange(2, 9)
        c["cached"] = _log_int(rng, 1, max(1, min(131072, int(4.0e8 / (row * c["B"])))))
    return c


# ---------------------------------------------------------------- sequences

def _batch(case):
    """(new tokens, cached tokens before them) of each sequence."""
    B, rng = case["B"], random.Random(case["mix"])
    if not case["ragged"]:
        return [case["new"]] * B, [case["cached"]] * B
    new = [1 if case["new"] == 1 else _log_int(rng, 1, case["new"]) for _ in range(B)]
    cached = [_log_int(rng, 1, case["cached"] + 1) - 1 for _ in range(B)]
    new[rng.randrange(B)] = case["new"]
    cached[rng.randrange(B)] = case["cached"]
    return new, cached


def _frequencies(rd, base, scaling, factor):
    """Turns' angles per position, 64 bits, and the factor on cosine and sine."""
    if scaling == "base":
        base = base * factor ** (rd / (rd - 2))
    f = torch.tensor([base ** (-2.0 * i / rd) for i in range(rd // 2)], dtype=torch.float64)
    if scaling == "linear":
        f = f / factor
    if scaling != "parts":
        return f, 1.0
    # unscaled above 32 turns within the original length, wholly scaled below one
    at = [rd * math.log(_ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
    low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rd - 1)
    ramp = ((torch.arange(rd // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
    return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0


_ORIGINAL = 32768  # the length that scaled frequencies were trained on


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    g, t = _gen(seed), _TYPES[case["x"]]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(t)
    s = {"case": case}
    if case["op"] == "rotate":
        T, heads, D = case["T"], case["heads"], case["D"]
        s["x"] = normal(T, heads * D + case["pad"])[:, :heads * D].unflatten(1, (heads, D))
        s["positions"] = torch.randint(0, case["far"], (T,), generator=g, device="cuda")
        rotary = (case["rd"], case["base"], case["layout"], case["scaling"], case["factor"])
    else:
        new, cached = _batch(case)
        B, Hq, Hkv, D, page = case["B"], case["Hq"], case["Hkv"], case["D"], case["page"]
        T, total = sum(new), [a + b for a, b in zip(new, cached)]
        pages = [-(-n // page) for n in total]
        count = sum(pages) + 3
        order = torch.randperm(count, generator=g, device="cuda").to(torch.int32)
        s["table"] = torch.full((B, max(pages)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(pages):
            s["table"][b, :n] = order[at:at + n]
            at += n
        s["k_cache"], s["v_cache"] = (normal(count, page, Hkv, D) for _ in range(2))
        s["lengths"] = torch.tensor(total, dtype=torch.int32, device="cuda")
        starts = [sum(new[:b]) for b in range(B + 1)]
        s["starts"] = None if case["new"] == 1 else torch.tensor(starts, dtype=torch.int32, device="cuda")
        s["host"] = (starts, total)  # a scheduler's own lists
        if case["op"] == "append":  # views of the rows of one projection
            qkv = normal(T, (Hq + 2 * Hkv) * D).unflatten(1, (Hq + 2 * Hkv, D))
            s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
            rotary = (case["rd"], 1.0e6, case["layout"], "none", 1.0)
        else:
            s["q"] = normal(T, Hq, D, std=2.0)
            rotary = None
    if own:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        import qmoe
        s["qmoe"] = qmoe
        if rotary:
            rd, base, layout, scaling, factor = rotary
            s["rotary"] = qmoe.Rotary(rd, base, layout=layout, scaling=None if scaling == "none" else scaling,
                                      factor=factor, original_length=_ORIGINAL, device="cuda")
    elif rotary:
        rd, base, layout, scaling, factor = rotary
        f, s["turn"] = _frequencies(rd, base, scaling, factor)
        s["frequencies"] = f.cuda()
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    case, q = s["case"], s["qmoe"]
    if case["op"] == "rotate":
        return q.rotate(s["x"], s["positions"], s["rotary"])
    if case["op"] == "append":
        turned = q.append_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], starts=s["starts"],
                             rotary=s["rotary"], q=s["q"])
        return turned, s["k_cache"], s["v_cache"]
    return q.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], starts=s["starts"],
                             window=case["window"])


def _turned(x, positions, frequencies, turn, layout):
    """x [T, heads, D] with its first 2 * len(frequencies) elements turned."""
    n = frequencies.shape[0]
    angle = positions.double()[:, None, None] * frequencies
    c, s = (torch.cos(angle) * turn).float(), (torch.sin(angle) * turn).float()
    v = x.float()
    out = v.clone()
    a, b = ((slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2)))
    out[..., a] = v[..., a] * c - v[..., b] * s
    out[..., b] = v[..., b] * c + v[..., a] * s
    return out.to(x.dtype)


def _places(s):
    """Position, page and place in it of every new token."""
    starts, total = s["host"]
    device, page = s["k_cache"].device, s["case"]["page"]
    seq = torch.cat([torch.full((starts[b + 1] - starts[b],), b, device=device) for b in range(len(total))])
    first = torch.tensor([total[b] - starts[b + 1] for b in range(len(total))], device=device)
    pos = torch.arange(seq.shape[0], device=device) + first[seq]
    return pos, s["table"][seq, pos // page].long(), pos % page


def _plain(s):
    case = s["case"]
    if case["op"] == "rotate":
        return _turned(s["x"], s["positions"], s["frequencies"], s["turn"], case["layout"])
    if case["op"] == "append":
        pos, page, place = _places(s)
        s["k_cache"][page, place] = _turned(s["k"], pos, s["frequencies"], s["turn"], case["layout"])
        s["v_cache"][page, place] = s["v"]
        return _turned(s["q"], pos, s["frequencies"], s["turn"], case["layout"]), s["k_cache"], s["v_cache"]
    starts, total = s["host"]
    Hkv, D, page, window = case["Hkv"], case["D"], case["page"], case["window"]
    G = case["Hq"] // Hkv
    out = torch.empty_like(s["q"])
    for b, n in enumerate(total):
        new = starts[b + 1] - starts[b]
        first = max(0, n - new - window + 1) // page * page if window else 0  # keys before it are out of every window
        pages = s["table"][b, first // page:-(-n // page)].long()
        keys = s["k_cache"][pages].flatten(0, 1)[:n - first]
        values = s["v_cache"][pages].flatten(0, 1)[:n - first]
        at = torch.arange(first, n, device=keys.device)
        row = torch.arange(n - new, n, device=keys.device).repeat_interleave(G)[:, None]
        seen = at <= row
        if window:
            seen = seen & (at > row - window)
        q = s["q"][starts[b]:starts[b + 1]].float().unflatten(1, (Hkv, G))
        for h in range(Hkv):
            score = torch.matmul(q[:, h].reshape(new * G, D), keys[:, h].float().t().contiguous()) * D ** -0.5
            score = torch.where(seen, score, float("-inf"))
            e = torch.exp(score - score.amax(dim=1, keepdim=True))
            o = torch.matmul(e, values[:, h].float()) / e.sum(dim=1, keepdim=True)
            out[starts[b]:starts[b + 1], h * G:(h + 1) * G] = o.view(new, G, D).to(out.dtype)
    return out


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = _BYTES[case["x"]]
    D = case["D"]
    if case["op"] == "rotate":
        n = case["T"] * case["heads"] * D
        return {"bytes": float(2 * n * size + 8 * case["T"]), "flops": 3.0 * case["T"] * case["heads"] * case["rd"]}
    new, cached = _batch(case)
    Hq, Hkv, T = case["Hq"], case["Hkv"], sum(new)
    if case["op"] == "append":
        return {"bytes": float(2 * T * (Hq + 2 * Hkv) * D * size), "flops": 3.0 * T * (Hq + Hkv) * case["rd"]}
    window = case["window"] or 1 << 60
    keys = pairs = 0
    for n, before in zip(new, cached):
        keys += min(before + n, n + window - 1)
        full = max(0, min(n, window - before - 1))  # rows whose window reaches the start
        pairs += full * before + full * (full + 1) // 2 + (n - full) * min(window, 1 << 50)
    return {"bytes": float(2 * T * Hq * D * size + 2 * keys * Hkv * D * size), "flops": 4.0 * pairs * Hq * D}


# ---------------------------------------------------------------- the same in 64 bits

def _exact_turn(x, pos, rd, base, layout, scaling="none", factor=1.0):
    i = torch.arange(rd // 2, dtype=torch.float64, device=x.device)
    length = 1.0
    if scaling == "base":
        base *= factor ** (rd / (rd - 2.0))
    w = torch.exp(-2.0 * i / rd * math.log(base))
    if scaling == "linear":
        w /= factor
    elif scaling == "parts":
        def index(turns):
            return rd / 2 * math.log(_ORIGINAL / (2 * math.pi * turns)) / math.log(base)
        low, high = max(0, math.floor(index(32))), min(rd - 1, math.ceil(index(1)))
        share = torch.clamp((i - low) / max(0.001, high - low), 0.0, 1.0)
        w *= 1.0 - share + share / factor
        length += 0.1 * math.log(factor)
    z = torch.polar(torch.full_like(w, length).expand(pos.shape[0], -1), pos.double().outer(w))[:, None]
    v = x.double()
    head, rest = v[..., :rd], v[..., rd:]
    if layout == "half":
        pair = torch.complex(*head.chunk(2, dim=-1)) * z
        return torch.cat([pair.real, pair.imag, rest], dim=-1)
    pair = torch.complex(head[..., 0::2].contiguous(), head[..., 1::2].contiguous()) * z
    return torch.cat([torch.view_as_real(pair).flatten(-2), rest], dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotate":
        return _exact_turn(s["x"], s["positions"], case["rd"], case["base"], case["layout"], case["scaling"],
                           case["factor"])
    new, cached = _batch(case)
    page, Hkv, at = case["page"], case["Hkv"], 0
    if case["op"] == "append":
        k_cache, v_cache, q = s["k_cache"].double(), s["v_cache"].double(), []
        for b, (n, before) in enumerate(zip(new, cached)):
            pos = torch.arange(before, before + n, device=s["q"].device)
            slot = s["table"][b].long()[pos // page] * page + pos % page
            k = _exact_turn(s["k"][at:at + n], pos, case["rd"], 1.0e6, case["layout"])
            k_cache.flatten(0, 1).index_copy_(0, slot, k)
            v_cache.flatten(0, 1).index_copy_(0, slot, s["v"][at:at + n].double())
            q.append(_exact_turn(s["q"][at:at + n], pos, case["rd"], 1.0e6, case["layout"]))
            at += n
        return torch.cat(q), k_cache, v_cache
    rows = []
    for b, (n, before) in enumerate(zip(new, cached)):
        pos = torch.arange(before + n, device=s["q"].device)
        slot = s["table"][b].long()[pos // page] * page + pos % page
        keys = s["k_cache"].flatten(0, 1)[slot]
        values = s["v_cache"].flatten(0, 1)[slot]
        step = max(1, 2 ** 25 // (before + n))
        for a in range(0, n, step):
            q = s["q"][at + a:at + min(n, a + step)].double()
            distance = (pos[before + a:before + a + q.shape[0], None] - pos)
            out = (distance < 0) | (distance >= (case["window"] or 1 << 60))
            heads = []
            for h in range(case["Hq"]):
                kv = h // (case["Hq"] // Hkv)
                p = q[:, h] @ keys[:, kv].double().t().contiguous() / math.sqrt(case["D"])
                heads.append(torch.softmax(p.masked_fill_(out, -math.inf), 1) @ values[:, kv].double())
            rows.append(torch.stack(heads, 1))
        at += n
    return torch.cat(rows)
