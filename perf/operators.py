"""Timed cases of the operators around the MoE block and after the lm_head.

* ``block_norm``: the RMS norm before a block;
* ``block_residual``: what follows a block: its norm, gate and residual scale, the
  residual sum, and the next block's norm of that sum;
* ``token_logprobs``: log probabilities of given tokens, entropy and top alternatives
  of a row of logits.

Hidden sizes are the ones of this repository's configurations (2048, 2560) and generic
ones, vocabularies generic; token counts go from one decoding sequence over a batch of
them to a long prefill. All of it is called eagerly.

Inputs are made on the device from the seed: block outputs N(0, 0.5), a residual stream
N(0, 2) with a few channels twenty times as wide, norm weights 1 + N(0, 0.1) (N(0, 0.1)
where the weight is stored as its distance from one), gates N(0, 1); logits N(0, 2.5)
with eight raised tokens per row, of which the given tokens are mostly one.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parent.parent / "qwen-ascend_amd")
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one decoding sequence: the norm before a block (the smallest call)
        {"name": "norm_b1", "op": "norm", "T": 1, "H": 2048, "x": "bf16", "out": "bf16", "w": "bf16", "offset": 0.0,
         "pad": 0},
        # the same over a prefill chunk
        {"name": "norm_t4096", "op": "norm", "T": 4096, "H": 2560, "x": "bf16", "out": "bf16", "w": "bf16",
         "offset": 0.0, "pad": 0},
        # a 32-bit residual stream normed to the block's 16 bits; rows are a slice of wider
        # rows, sizes are odd, weights are stored as their distance from one
        {"name": "norm_stream_ragged", "op": "norm", "T": 777, "H": 1999, "x": "fp32", "out": "bf16", "w": "fp32",
         "offset": 1.0, "pad": 9},
        # a few sequences decoding together: the whole step after a block
        {"name": "residual_b4", "op": "residual", "T": 4, "H": 2560, "y": "bf16", "res": "bf16", "w": "bf16",
         "post": True, "gate": "row", "sigmoid": True, "scale": 1.0, "next": True, "offset": 0.0},
        # the same over a prefill chunk
        {"name": "residual_t4096", "op": "residual", "T": 4096, "H": 2560, "y": "bf16", "res": "bf16", "w": "bf16",
         "post": True, "gate": "row", "sigmoid": True, "scale": 1.0, "next": True, "offset": 0.0},
        # a long prefill over a 32-bit stream, a gate per channel and a residual scale
        {"name": "residual_stream_t8192", "op": "residual", "T": 8192, "H": 4096, "y": "bf16", "res": "fp32",
         "w": "fp32", "post": False, "gate": "channel", "sigmoid": False, "scale": 0.22, "next": True, "offset": 1.0},
        # half precision at odd sizes, a gate per element, the last block (no norm after it)
        {"name": "residual_odd_fp16", "op": "residual", "T": 1003, "H": 2047, "y": "fp16", "res": "fp16", "w": "fp16",
         "post": True, "gate": "full", "sigmoid": True, "scale": 0.5, "next": False, "offset": 0.0},
        # one decoding sequence: its token's log probability and twenty alternatives
        {"name": "logprobs_b1", "op": "logprobs", "T": 1, "V": 131072, "x": "bf16", "m": 1, "top": 20, "allowed": "none"},
        # a batch of decoding sequences under a grammar: a mask of allowed tokens for each
        {"name": "logprobs_b48_allowed", "op": "logprobs", "T": 48, "V": 131072, "x": "bf16", "m": 1, "top": 8,
         "allowed": "rows"},
        # the loss of a prompt chunk: no alternatives (the largest case)
        {"name": "logprobs_t4096", "op": "logprobs", "T": 4096, "V": 131072, "x": "bf16", "m": 1, "top": 0,
         "allowed": "none"},
        # scoring a chunk with alternatives from 32-bit logits
        {"name": "logprobs_t1024_top20", "op": "logprobs", "T": 1024, "V": 65536, "x": "fp32", "m": 1, "top": 20,
         "allowed": "none"},
        # several candidates for each row, odd sizes, rows that start off any alignment
        {"name": "logprobs_candidates_odd", "op": "logprobs", "T": 333, "V": 50003, "x": "fp16", "m": 4, "top": 5,
         "allowed": "vocabulary"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "residual", "logprobs"))
    t = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "logprobs":
        V = _log_int(rng, 1000, 160000)
        allowed = rng.choice(("none", "none", "rows", "vocabulary"))
        most = int(1.0e9 / (V * (_BYTES[t] + (1 if allowed == "rows" else 0))))
        return {"op": op, "T": _log_int(rng, 1, min(most, 4096)), "V": V, "x": t, "m": rng.choice((1, 1, 1, 2, 5)),
                "top": rng.choice((0, 1, 5, 8, 20)), "allowed": allowed}
    H = _log_int(rng, 64, 16384)
    if rng.random() < 0.5:
        H = -(-H // 64) * 64
    T = _log_int(rng, 1, min(16384, int(4.0e7 / H)))
    w = rng.choice((t, "fp32"))
    offset = rng.choice((0.0, 1.0))
    if op == "norm":
        wide = t != "fp32" and rng.random() < 0.3
        return {"op": op, "T": T, "H": H, "x": "fp32" if wide else t, "out": t, "w": w, "offset": offset,
                "pad": rng.choice((0, 0, 8, 5))}
    post = rng.random() < 0.6
    return {"op": op, "T": T, "H": H, "y": t, "res": "fp32" if rng.random() < 0.3 else t, "w": w, "post": post,
            "gate": rng.choice(("none", "row", "channel", "full")), "sigmoid": rng.random() < 0.5,
            "scale": rng.choice((1.0, 0.22, 0.5)), "next": not post or rng.random() < 0.7, "offset": offset}


# ---------------------------------------------------------------- inputs

def _normal(g, shape, std, dtype):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(_TYPES[dtype])


def _stream(g, T, H, dtype):
    wide = torch.where(torch.rand(H, generator=g, device="cuda") < 0.004, 20.0, 1.0)
    return (torch.randn((T, H), generator=g, device="cuda") * 2.0 * wide).to(_TYPES[dtype])


def _weight(g, H, dtype, offset):
    return (1.0 - offset + 0.1 * torch.randn(H, generator=g, device="cuda")).to(_TYPES[dtype])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "norm":
        T, H = case["T"], case["H"]
        s["x"] = _stream(g, T, H + case["pad"], case["x"])[:, :H]
        s["w"] = _weight(g, H, case["w"], case["offset"])
    elif case["op"] == "residual":
        T, H = case["T"], case["H"]
        s["y"] = _normal(g, (T, H), 0.5, case["y"])
        s["res"] = _stream(g, T, H, case["res"])
        s["post"] = _weight(g, H, case["w"], case["offset"]) if case["post"] else None
        s["next"] = _weight(g, H, case["w"], case["offset"]) if case["next"] else None
        shape = {"none": None, "row": (T, 1), "channel": (H,), "full": (T, H)}[case["gate"]]
        s["gate"] = None if shape is None else _normal(g, shape, 1.0, case["y"])
    else:
        T, V, m = case["T"], case["V"], case["m"]
        x = torch.randn((T, V), generator=g, device="cuda").mul_(2.5)
        raised = torch.randint(0, V, (T, 8), generator=g, device="cuda")
        x.scatter_add_(1, raised, 4.0 + 8.0 * torch.rand((T, 8), generator=g, device="cuda"))
        s["x"] = x.to(_TYPES[case["x"]])
        del x
        pick = torch.randint(0, 8, (T, m), generator=g, device="cuda")
        other = torch.randint(0, V, (T, m), generator=g, device="cuda")
        likely = torch.rand((T, m), generator=g, device="cuda") < 0.8
        s["tokens"] = torch.where(likely, raised.gather(1, pick), other)
        s["allowed"] = None
        if case["allowed"] == "vocabulary":  # a padded or reserved part of the vocabulary
            s["allowed"] = torch.rand(V, generator=g, device="cuda") < 0.98
            s["allowed"][s["tokens"].reshape(-1)] = True
        elif case["allowed"] == "rows":      # between a tenth and all of the tokens
            share = 0.1 + 0.9 * torch.rand((T, 1), generator=g, device="cuda")
            s["allowed"] = torch.rand((T, V), generator=g, device="cuda") < share
            s["allowed"].scatter_(1, s["tokens"], True)
    if own:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        import qmoe
        s["qmoe"] = qmoe
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    case, q = s["case"], s["qmoe"]
    if case["op"] == "norm":
        return q.block_norm(s["x"], s["w"], offset=case["offset"], out_dtype=_TYPES[case["out"]])
    if case["op"] == "residual":
        return q.block_residual(s["y"], s["res"], post_weight=s["post"], gate=s["gate"],
                                gate_act="sigmoid" if case["sigmoid"] and s["gate"] is not None else None,
                                scale=case["scale"], next_weight=s["next"], offset=case["offset"])
    r = q.token_logprobs(s["x"], s["tokens"], top=case["top"], allowed=s["allowed"])
    if not case["top"]:
        return r.logprobs, r.entropy
    return r.logprobs, r.entropy, r.top_ids, r.top_logprobs


def _rms(v, w, offset):
    r = torch.rsqrt((v * v).mean(dim=1, keepdim=True) + 1e-6)
    return v * r * (offset + w.float())


def _plain(s):
    case = s["case"]
    if case["op"] == "norm":
        return _rms(s["x"].float(), s["w"], case["offset"]).to(_TYPES[case["out"]])
    if case["op"] == "residual":
        y = s["y"].float()
        if s["post"] is not None:
            y = _rms(y, s["post"], case["offset"])
        if s["gate"] is not None:
            gate = s["gate"].float()
            if case["sigmoid"]:
                gate = 1.0 / (1.0 + torch.exp(-gate))
            y = y * gate
        h = s["res"].float() + case["scale"] * y
        stream = h.to(s["res"].dtype)
        if s["next"] is None:
            return stream
        return stream, _rms(h, s["next"], case["offset"]).to(s["y"].dtype)
    x, top = s["x"].float(), case["top"]
    if s["allowed"] is not None:
        x = torch.where(s["allowed"], x, float("-inf"))
    shifted = x - x.amax(dim=1, keepdim=True)
    e = torch.exp(shifted)
    total = e.sum(dim=1, keepdim=True)
    logtotal = torch.log(total)
    weighted = (e * torch.where(e > 0, shifted, 0.0)).sum(dim=1, keepdim=True)
    entropy = (logtotal - weighted / total).squeeze(1)
    logprobs = shifted.gather(1, s["tokens"]) - logtotal
    if not top:
        return logprobs, entropy
    # distinct whole numbers in the order of (logit, lower id first)
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    ids = torch.arange(x.shape[1], device=x.device)
    best = torch.topk((order << 32) + (0x7FFFFFFF - ids), top, dim=1)[0]
    top_ids = 0x7FFFFFFF - (best & 0xFFFFFFFF)
    return logprobs, entropy, top_ids, shifted.gather(1, top_ids) - logtotal


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    T = case["T"]
    if case["op"] == "norm":
        H = case["H"]
        return {"bytes": float(T * H * (_BYTES[case["x"]] + _BYTES[case["out"]]) + H * _BYTES[case["w"]]),
                "flops": 4.0 * T * H}
    if case["op"] == "residual":
        H, y = case["H"], _BYTES[case["y"]]
        b = T * H * (y + 2 * _BYTES[case["res"]] + (y if case["next"] else 0))
        b += H * _BYTES[case["w"]] * (case["post"] + case["next"])
        b += {"none": 0, "row": T, "channel": H, "full": T * H}[case["gate"]] * y
        return {"bytes": float(b), "flops": T * H * (3.0 + 4.0 * case["post"] + 4.0 * case["next"])}
    V = case["V"]
    b = T * V * _BYTES[case["x"]] + {"none": 0, "rows": T * V, "vocabulary": V}[case["allowed"]]
    b += T * (case["m"] * 12 + 4 + case["top"] * 12)
    return {"bytes": float(b), "flops": 6.0 * T * V}


# ---------------------------------------------------------------- the same in 64 bits

def _exact_norm(v, w, offset):
    ms = v.square().sum(-1, keepdim=True) / v.shape[-1]
    return v / (ms + 1e-6).sqrt() * (w.double() + offset)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s["x"].double(), s["w"], case["offset"])
    if case["op"] == "residual":
        block = s["y"].double()
        if case["post"]:
            block = _exact_norm(block, s["post"], case["offset"])
        if case["gate"] != "none":
            gate = s["gate"].double()
            block = (gate.sigmoid() if case["sigmoid"] else gate) * block
        h = s["res"].double() + block * case["scale"]
        return (h, _exact_norm(h, s["next"], case["offset"])) if case["next"] else h
    out = ([], [], [], [])
    rows = max(1, 2 ** 25 // case["V"])
    for a in range(0, case["T"], rows):
        x = s["x"][a:a + rows].double()
        if s["allowed"] is not None:
            mask = s["allowed"] if s["allowed"].dim() == 1 else s["allowed"][a:a + rows]
            x.masked_fill_(~mask, -math.inf)
        logp = x - torch.logsumexp(x, 1, keepdim=True)
        out[0].append(logp.gather(1, s["tokens"][a:a + rows]))
        out[1].append(-(logp.exp() * logp).nan_to_num_(nan=0.0).sum(1))
        if case["top"]:
            ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :case["top"]]
            out[2].append(ids)
            out[3].append(logp.gather(1, ids))
    return tuple(torch.cat(o) for o in out if o)
