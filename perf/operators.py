"""The operators that are measured: cases, inputs, plain forms and their exact values.

Three operators of the transformer block around the INT8 linear layers:

* ``rms``  residual addition, RMS norm and an 8-bit output with one scale a row
  (``h3_speedkit.ops.rms_quant.residual_rms_quant``), the input of an INT8 linear;
* ``rope`` rotary positions with several axes, with the per-head RMS norm of Q and K
  where it is given (``h3_speedkit.ops.rope.rope_axes``), and the table of rotations
  that the QKV op takes (``rope_table``);
* ``attn`` attention under document, padding, causal and prefix masks, with scores
  capped by a tanh and a bias by distance
  (``h3_speedkit.ops.masked_attention.masked_attention``).

``run`` computes their plain forms from elementary torch operations, or calls the
framework where ``own`` is true.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one token's hidden row into the QKV projection: latency
        dict(name="rms token", op="rms", rows=1, width=4096, type="bf16", codes="int8", residual=True),
        # the H3 hidden width over 16384 tokens, residual stream updated on the way
        dict(name="rms block", op="rms", rows=16384, width=5376, type="bf16", codes="int8", residual=True),
        # an odd width (no vector loads), FP16, no residual, 8-bit floating codes
        dict(name="rms odd", op="rms", rows=1999, width=1155, type="fp16", codes="e4m3", residual=False),
        # Q and K of one token, 56 heads, normalised per head, 96 of 128 channels rotated
        dict(name="rope token", op="rope", tokens=1, q_heads=56, k_heads=56, dim=128, axes="16,16,16", type="bf16",
             norm=True, split=True, whole=True),
        # a video's tokens (time, height, width), the same heads
        dict(name="rope video", op="rope", tokens=16384, q_heads=56, k_heads=56, dim=128, axes="16,16,16", type="bf16",
             norm=True, split=True, whole=True),
        # fractional positions, adjacent pairs, an odd number of pairs, grouped heads
        dict(name="rope odd", op="rope", tokens=3001, q_heads=24, k_heads=8, dim=64, axes="7,9,11", type="fp16",
             norm=False, split=False, whole=False),
        # the table of 48 rotations a token that the QKV op reads, for 98304 tokens
        dict(name="rope table", op="table", tokens=98304, axes="16,16,16", whole=True),
        # one query a sequence over long keys: a pooled token, or one new token
        dict(name="attn single", op="attn", batch=2, queries=1, keys=32768, q_heads=56, k_heads=8, dim=128, type="bf16",
             documents=0, padded=False, causal=False, prefix=0, cap=0.0, distance=False),
        # every token with every token: a video's block without masks
        dict(name="attn dense", op="attn", batch=1, queries=8192, keys=8192, q_heads=24, k_heads=24, dim=128,
             type="bf16", documents=0, padded=False, causal=False, prefix=0, cap=0.0, distance=False),
        # packed documents of ragged lengths (some empty, some of one token), grouped heads
        dict(name="attn documents", op="attn", batch=1, queries=12288, keys=12288, q_heads=16, k_heads=4, dim=128,
             type="bf16", documents=21, padded=False, causal=False, prefix=0, cap=0.0, distance=False),
        # a prompt that sees itself whole, then causal, scores capped
        dict(name="attn prefix", op="attn", batch=1, queries=6000, keys=6000, q_heads=8, k_heads=2, dim=128,
             type="bf16", documents=0, padded=False, causal=True, prefix=700, cap=30.0, distance=False),
        # a padded batch of prompts, bias by distance, 64 channels a head
        dict(name="attn distance", op="attn", batch=5, queries=333, keys=333, q_heads=12, k_heads=12, dim=64,
             type="fp16", documents=0, padded=True, causal=False, prefix=0, cap=0.0, distance=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("rms", "rope", "table", "attn", "attn"))
    kind = rng.choice(("bf16", "fp16"))
    if op == "rms":
        width = _log_int(rng, 64, 8192)
        if rng.random() < 0.6:
            width = (width + 15) // 16 * 16
        return dict(op=op, rows=_log_int(rng, 1, 10000), width=width, type=kind, codes=rng.choice(("int8", "e4m3")),
                    residual=rng.random() < 0.7)
    if op in ("rope", "table"):
        n = rng.randint(1, 3)
        axes = [rng.randint(1, 64 // n) for _ in range(n)]
        if rng.random() < 0.6:
            axes = [a // 8 * 8 or 8 for a in axes]
        text, whole = ",".join(map(str, axes)), rng.random() < 0.5
        if op == "table":
            return dict(op=op, tokens=_log_int(rng, 1, 98304), axes=text, whole=whole)
        return dict(op=op, tokens=_log_int(rng, 1, 8192), q_heads=rng.randint(1, 48), k_heads=rng.randint(1, 48),
                    dim=128 if sum(axes) > 32 else rng.choice((64, 128)), axes=text, type=kind,
                    norm=rng.random() < 0.5, split=rng.random() < 0.5, whole=whole)
    k_heads = rng.randint(1, 6)
    group, dim = rng.choice((1, 1, 2, 3, 4, 7)), rng.choice((64, 128))
    form = rng.choice(("single", "square", "documents", "padded"))
    case = dict(op=op, batch=1, q_heads=k_heads * group, k_heads=k_heads, dim=dim, type=kind, documents=0, padded=False,
                causal=rng.random() < 0.5, prefix=0, cap=rng.choice((0.0, 0.0, 20.0, 50.0)),
                distance=rng.random() < 0.4)
    if form == "single":
        case.update(batch=rng.randint(1, 4), queries=_log_int(rng, 1, 16), keys=_log_int(rng, 16, 32768))
    elif form == "square":
        n = _log_int(rng, 64, 5000)
        case.update(queries=n, keys=n)
    elif form == "documents":
        n = _log_int(rng, 64, 6000)
        case.update(queries=n, keys=n, documents=rng.randint(2, 30))
    else:
        n = _log_int(rng, 16, 1500)
        case.update(batch=rng.randint(2, 5), queries=n, keys=n, padded=True)
    if case["causal"] and rng.random() < 0.6:
        case["prefix"] = rng.randint(1, 800)
    return case


# ---- the ranges of an attention case, as plain numbers -----------------------------------

def _offsets(case):
    """Where packed documents begin and end: ragged, the first two of no and of one token."""
    n, total = case["documents"], case["queries"]
    rng = random.Random(1000 * n + total)
    cuts = sorted(rng.randint(1, total) for _ in range(n - 3)) if n > 3 else []
    return ([0, 0, 1] + cuts + [total])[: n] + [total]


def _lengths(case):
    """The valid tokens of each sequence of a padded batch: the first whole, the last of one."""
    rng = random.Random(case["queries"] + case["batch"])
    n = [rng.randint(1, case["queries"]) for _ in range(case["batch"])]
    return [case["queries"]] + n[1:-1] + [1]


def _visible(case):
    """(query, key) pairs that are not masked, over the batch, for one head."""
    if case["documents"]:
        o = _offsets(case)
        spans = [(b - a, b - a) for a, b in zip(o, o[1:])]
    elif case["padded"]:
        spans = [(n, n) for n in _lengths(case)]
    else:
        spans = [(case["queries"], case["keys"])] * case["batch"]
    if not case["causal"]:
        return sum(a * b for a, b in spans)
    p = case["prefix"]
    return sum(sum(min(k, max(p, i + 1 + k - q, 0)) for i in range(q)) for q, k in spans)


def work(case):
    if case["op"] == "rms":
        n = case["rows"] * case["width"]
        return {"bytes": n * (7 if case["residual"] else 3) + 4 * case["rows"] + 2 * case["width"], "flops": 6 * n}
    pairs = sum(map(int, case["axes"].split(","))) if "axes" in case else 0
    if case["op"] == "table":
        return {"bytes": case["tokens"] * (8 * pairs + 4 * len(case["axes"].split(","))),
                "flops": 20 * case["tokens"] * pairs}
    if case["op"] == "rope":
        n = case["tokens"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        return {"bytes": 4 * n + 4 * case["tokens"] * len(case["axes"].split(",")), "flops": (7 if case["norm"] else 3) * n}
    tokens = case["batch"] * case["queries"] * case["q_heads"], case["batch"] * case["keys"] * case["k_heads"]
    return {"bytes": 4 * case["dim"] * sum(tokens) + 4 * tokens[0],
            "flops": 4 * case["dim"] * case["q_heads"] * _visible(case)}


# ---- inputs ---------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, like=torch.float32, by=1.0):
        return (torch.randn(shape, generator=g, device=dev) * by).to(like)

    state = dict(case=case)
    if case["op"] == "rms":
        t, shape = TYPES[case["type"]], (case["rows"], case["width"])
        state.update(x=normal(*shape, like=t), residual=normal(*shape, like=t, by=3.0) if case["residual"] else None,
                     weight=(1 + normal(case["width"], by=0.2)).to(t))
        return state
    if case["op"] in ("rope", "table"):
        axes = tuple(map(int, case["axes"].split(",")))
        # a grid's coordinates: frames few, rows and columns more; or text far along one line
        far = torch.tensor([4000, 90, 160][: len(axes)], device=dev)
        at = torch.rand((case["tokens"], len(axes)), generator=g, device=dev) * far
        state.update(positions=at.floor().to(torch.int32) if case["whole"] else at, axes=axes)
        if case["op"] == "rope":
            t, d = TYPES[case["type"]], case["dim"]
            # Q, K and V lie side by side in one projection's rows
            qkv = normal(case["tokens"], (case["q_heads"] + 2 * case["k_heads"]) * d, like=t)
            a, b = case["q_heads"] * d, (case["q_heads"] + case["k_heads"]) * d
            state.update(q=qkv[:, :a].view(case["tokens"], -1, d), k=qkv[:, a:b].view(case["tokens"], -1, d))
            state.update({n: (1 + normal(d, by=0.2)).to(t) if case["norm"] else None for n in ("q_weight", "k_weight")})
        return state
    t, b, d = TYPES[case["type"]], case["batch"], case["dim"]
    state.update(q=normal(b, case["queries"], case["q_heads"], d, like=t, by=2.0),
                 k=normal(b, case["keys"], case["k_heads"], d, like=t),
                 v=normal(b, case["keys"], case["k_heads"], d, like=t))
    # the rows behind a padded batch's sequences stay as they are in these
    state["out"] = torch.zeros_like(state["q"])
    state["lse"] = torch.zeros((b, case["q_heads"], case["queries"]), device=dev)
    ints = dict(device=dev, dtype=torch.int32)
    state["offsets"] = torch.tensor(_offsets(case), **ints) if case["documents"] else None
    state["lengths"] = torch.tensor(_lengths(case), **ints) if case["padded"] else None
    groups = case["documents"] or b
    state["prefix"] = torch.full((groups,), case["prefix"], **ints) if case["prefix"] else None
    heads = torch.arange(1, case["q_heads"] + 1, device=dev)
    state["slopes"] = torch.exp2(-8.0 * heads / case["q_heads"]) if case["distance"] else None
    return state


# ---- one pass ---------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


EPS, THETA = 1e-6, 10000.0


def _plain_rms(s):
    t = s["x"].dtype
    h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(t)
    f = h.float()
    y = f * torch.rsqrt((f * f).mean(1, keepdim=True) + EPS) * s["weight"].float()
    top = 127.0 if s["case"]["codes"] == "int8" else 448.0
    scale = (y.abs().amax(1, keepdim=True) / top).clamp_min(1e-30)
    codes = y / scale
    codes = codes.round() if top == 127.0 else codes.clamp(-448, 448).to(torch.float8_e4m3fn).float()
    return {"values": (codes * scale).to(t), "scale": scale, "sum": h}


def _angles(s):
    """Each token's angles, in 64 bits: far positions lose theirs in 32."""
    at = s["positions"].double()
    angles = [at[:, a:a + 1] * THETA ** -(torch.arange(n, device=at.device, dtype=torch.float64) / n)
              for a, n in enumerate(s["axes"])]
    return torch.cat(angles, 1)


def _plain_turn(x, weight, angles, split):
    f, n = x.float(), angles.shape[1]
    if weight is not None:
        f = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * weight.float()
    c, si = torch.cos(angles).float()[:, None], torch.sin(angles).float()[:, None]
    if split:
        a, b = f[..., :n], f[..., n:2 * n]
        turned = torch.cat((a * c - b * si, b * c + a * si), -1)
    else:
        a, b = f[..., 0:2 * n:2], f[..., 1:2 * n:2]
        turned = torch.stack((a * c - b * si, b * c + a * si), -1).flatten(-2)
    return torch.cat((turned, f[..., 2 * n:]), -1).to(x.dtype)


def _plain_rope(s):
    angles, split = _angles(s), s["case"]["split"]
    return {"q": _plain_turn(s["q"], s["q_weight"], angles, split), "k": _plain_turn(s["k"], s["k_weight"], angles, split)}


def _plain_table(s):
    a = _angles(s)
    c, si = torch.cos(a), torch.sin(a)
    return torch.stack((c, -si, si, c), -1).view(1, a.shape[0], 1, a.shape[1], 2, 2).to(torch.bfloat16)


def _plain_attn(s):
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    b, nq, h, d = q.shape
    nk, hk = k.shape[1:3]
    q4 = q.float().permute(0, 2, 1, 3).reshape(b, hk, h // hk, nq, d)
    k4, v4 = (x.float().permute(0, 2, 1, 3)[:, :, None] for x in (k, v))
    score = torch.matmul(q4, k4.transpose(-1, -2)).view(b, h, nq, nk)
    score *= d ** -0.5
    if case["cap"]:
        score = torch.tanh(score / case["cap"]) * case["cap"]
    i, j = (torch.arange(n, device=q.device) for n in (nq, nk))
    if s["offsets"] is not None:
        o = s["offsets"].long()
        doc = (i[:, None] >= o[None, 1:]).sum(1)          # packed: queries and keys alike
        begin, qlen = o[doc], o[doc + 1] - o[doc]
        klen, prefix = qlen, None if s["prefix"] is None else s["prefix"].long()[doc]
        begin, qlen, klen = begin[None, :, None], qlen[None, :, None], klen[None, :, None]
        prefix = None if prefix is None else prefix[None, :, None]
    else:
        whole = torch.tensor([nq], device=q.device), torch.tensor([nk], device=q.device)
        qlen, klen = (s["lengths"].long(), s["lengths"].long()) if s["lengths"] is not None else whole
        begin, qlen, klen = torch.zeros_like(qlen)[:, None, None], qlen[:, None, None], klen[:, None, None]
        prefix = None if s["prefix"] is None else s["prefix"].long()[:, None, None]
    at = i[None, :, None] - begin + klen - qlen            # the query's place among its keys
    jl = j[None, None, :] - begin
    see = (jl >= 0) & (jl < klen)
    if case["causal"]:
        see = see & ((jl <= at) if prefix is None else (jl <= at) | (jl < prefix))
    if s["slopes"] is not None:
        score = score - s["slopes"][None, :, None, None] * (at - jl).abs().float()[:, None]
    score = score.masked_fill(~see[:, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top.clamp_min(-1e30))
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, 1.0)
    out = torch.matmul(p.view(b, hk, h // hk, nq, nk), v4).view(b, h, nq, d).permute(0, 2, 1, 3)
    lse = (top + torch.log(total))[..., 0]
    inside = ((i[None, :] < qlen[..., 0]) if s["lengths"] is not None else torch.ones_like(i, dtype=torch.bool)[None])
    s["out"].copy_(torch.where(inside[:, :, None, None], out, 0.0))
    s["lse"].copy_(torch.where(inside[:, None], lse, 0.0))
    return {"out": s["out"], "lse": s["lse"]}


_PLAIN = {"rms": _plain_rms, "rope": _plain_rope, "table": _plain_table, "attn": _plain_attn}


def _framework():
    path = str(Path(__file__).resolve().parents[1] / "comfyui-h3-speedkit_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from h3_speedkit.ops import masked_attention, rms_quant, rope
    return masked_attention, rms_quant, rope


def _own_rms(s):
    codes, scale, h = _framework()[1].residual_rms_quant(
        s["x"], s["weight"], residual=s["residual"], eps=EPS,
        dtype=torch.int8 if s["case"]["codes"] == "int8" else torch.float8_e4m3fn)
    return {"values": (codes.float() * scale).to(s["x"].dtype), "scale": scale, "sum": h}


def _own_rope(s):
    q, k = _framework()[2].rope_axes(s["q"], s["k"], s["positions"], sections=s["axes"], theta=THETA,
                                     interleaved=not s["case"]["split"], q_weight=s["q_weight"],
                                     k_weight=s["k_weight"], eps=EPS)
    return {"q": q, "k": k}


def _own_table(s):
    return _framework()[2].rope_table(s["positions"], sections=s["axes"], theta=THETA)


def _own_attn(s):
    case = s["case"]
    out, lse = _framework()[0].masked_attention(
        s["q"], s["k"], s["v"], softcap=case["cap"], slopes=s["slopes"], causal=case["causal"], prefix=s["prefix"],
        q_offsets=s["offsets"], k_offsets=s["offsets"], q_lengths=s["lengths"], k_lengths=s["lengths"], out=s["out"],
        lse=s["lse"])
    return {"out": out, "lse": lse}


_OWN = {"rms": _own_rms, "rope": _own_rope, "table": _own_table, "attn": _own_attn}


# ---- exact values: the definitions in 64 bits, written on their own ------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["op"]](s)


def _round_e4m3(v):
    """The nearest value with three bits behind the point and exponents from -6, ties to even."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -20))).clamp_min(-6.0)
    step = torch.exp2(e - 3)
    return torch.round(v / step) * step


def _exact_rms(s):
    h = s["x"].double()
    if s["residual"] is not None:
        h = h + s["residual"].double()
        h = h.to(s["x"].dtype).double()                   # the stream is stored in its type
    norm = h / torch.sqrt(h.pow(2).sum(1, keepdim=True) / h.shape[1] + EPS) * s["weight"].double()[None]
    whole = s["case"]["codes"] == "int8"
    scale = torch.clamp(norm.abs().max(1, keepdim=True).values / (127 if whole else 448), min=1e-30)
    codes = torch.round(norm / scale) if whole else _round_e4m3(norm / scale)
    return {"values": codes * scale, "scale": scale, "sum": h}


def _exact_turn(s, x, weight):
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * weight.double()
    y, pair, pairs = x.clone(), 0, sum(s["axes"])
    for axis, n in enumerate(s["axes"]):
        for i in range(n):
            turn = s["positions"][:, axis].double() / THETA ** (i / n)
            a, b = (pair, pairs + pair) if s["case"]["split"] else (2 * pair, 2 * pair + 1)
            z = torch.complex(x[:, :, a], x[:, :, b]) * torch.polar(torch.ones_like(turn), turn)[:, None]
            y[:, :, a], y[:, :, b] = z.real, z.imag
            pair += 1
    return y


def _exact_rope(s):
    return {"q": _exact_turn(s, s["q"], s["q_weight"]), "k": _exact_turn(s, s["k"], s["k_weight"])}


def _exact_table(s):
    rows = []
    for axis, n in enumerate(s["axes"]):
        for i in range(n):
            z = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"),
                            s["positions"][:, axis].double() / THETA ** (i / n))
            rows.append(torch.stack((z.real, -z.imag, z.imag, z.real), -1).view(-1, 2, 2))
    return torch.stack(rows, 1)[None, :, None]


def _exact_attn(s):
    case, (b, nq, h, d) = s["case"], s["q"].shape
    nk, group = s["k"].shape[1], h // s["k"].shape[2]
    out = torch.zeros((b, nq, h, d), dtype=torch.float64, device="cuda")
    lse = torch.zeros((b, h, nq), dtype=torch.float64, device="cuda")
    if case["documents"]:
        o = _offsets(case)
        parts = [(0, a, z, a, z, n) for n, (a, z) in enumerate(zip(o, o[1:]))]
    elif case["padded"]:
        parts = [(n, 0, z, 0, z, n) for n, z in enumerate(_lengths(case))]
    else:
        parts = [(n, 0, nq, 0, nk, n) for n in range(b)]
    for n, a, z, ka, kz, _ in parts:
        if z == a:
            continue
        far = torch.arange(z - a, device="cuda")[:, None] + (kz - ka) - (z - a) - torch.arange(kz - ka, device="cuda")
        hidden = (far < 0) & (torch.arange(kz - ka, device="cuda") >= case["prefix"]) if case["causal"] else None
        for head in range(h):
            x = s["q"][n, a:z, head].double() @ s["k"][n, ka:kz, head // group].double().T / math.sqrt(d)
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["distance"]:
                x = x - s["slopes"][head].double() * far.abs()
            if hidden is not None:
                x = x.masked_fill(hidden, -math.inf)
            total = torch.logsumexp(x, 1)
            lse[n, head, a:z] = total
            weight = torch.exp(x - total[:, None])
            out[n, a:z, head] = torch.where(torch.isfinite(total)[:, None], weight, 0.0) @ s["v"][n, ka:kz, head // group].double()
    return {"out": out, "lse": lse}


_EXACT = {"rms": _exact_rms, "rope": _exact_rope, "table": _exact_table, "attn": _exact_attn}
