"""Operands of the INT8 block's golden cases, from integer arithmetic alone (the same on
every host and with every version of a random generator), and their outputs."""
import numpy as np
import torch


def mixed(seed, *shape):
    """Whole numbers of 0 .. 2^24 - 1, a multiplicative hash of the element's number."""
    n = np.arange(int(np.prod(shape)), dtype=np.uint64) + np.uint64(seed) * np.uint64(1000003)
    for _ in range(2):
        n = ((n ^ (n >> np.uint64(31))) * np.uint64(0x9E3779B97F4A7C15)) & np.uint64(0xFFFFFFFFFFFFFFFF)
    return (n >> np.uint64(40)).astype(np.int64).reshape(shape)


def codes(seed, *shape):
    return torch.from_numpy((mixed(seed, *shape) % 255 - 127).astype(np.int8))


def between(seed, low, high, *shape):
    """FP32 between low and high."""
    return torch.from_numpy((low + (high - low) * (mixed(seed, *shape) / 2.0 ** 24)).astype(np.float32))


# tokens, heads, K/V heads, spread of the scores, first block of 128 queries
ATTENTION = {"ragged": (300, 1, 1, 1.0, 0), "grouped": (129, 4, 2, 8.0, 0), "window": (256, 2, 1, 0.05, 1)}
# tokens, heads, hidden width; whether the rows share an offset and hardly turn (anchors fire)
QKV = {"few": (130, 2, 256, False), "many": (300, 1, 256, True)}


def attention(name, device):
    """Packed operands of the INT8 attention, and the first query block."""
    from h3_speedkit.ops.qkv import PrequantizedInt8Attention
    m, heads, kv_heads, spread, start = ATTENTION[name]
    parts = (m + 127) // 128
    t = dict(q=codes(1, 1, heads, m, 128), k=codes(2, 1, kv_heads, m, 128), v=codes(3, kv_heads * 128, parts * 128),
             q_scale=between(4, 0.001, 0.021, 1, heads, parts * 32) * spread,
             k_scale=between(5, 0.001, 0.021, 1, kv_heads, parts * 4) * spread,
             v_scale=between(6, 0.0005, 0.0105, kv_heads * 128))
    return PrequantizedInt8Attention(**{n: x.to(device) for n, x in t.items()}, original_head_dim=128,
                                     input_dtype=torch.bfloat16, attention_scale=128 ** -0.5, cta_k=128,
                                     attn_mask=None), start


def run_attention(name, device):
    from h3_speedkit.ops.dense import DenseLibrary, allocate_output
    packed, start = attention(name, device)
    out = allocate_output(packed, "bshd")
    DenseLibrary().bind(packed, out, start=start)()
    return {"out": out.contiguous().view(torch.int16)}


def run_qkv(name, device):
    from h3_speedkit.ops.qkv import QKV as Op
    m, heads, hidden, offset = QKV[name]
    q, rope = codes(11, m, hidden), between(16, -1.0, 1.0, 1, m, 1, 48, 2, 2)
    if offset:
        q = (q.int() // 10 + torch.from_numpy(mixed(12, 1, hidden) % 109 - 54).int()).to(torch.int8)
        rope = torch.tensor([[1.0, 0.0], [0.0, 1.0]]) + rope * torch.tensor([[0.0, 0.05], [0.05, 0.0]])
    args = (q, codes(13, 3 * heads * 128, hidden), between(14, 0.001, 0.01, m, 1),
            between(15, 0.0005, 0.005, 3 * heads * 128, 1), rope.bfloat16(),
            between(17, 0.5, 1.5, 128).bfloat16(), between(18, 0.5, 1.5, 128).bfloat16())
    out = Op().run(*(t.to(device) for t in args), 1e-6, heads=heads)
    return {n: out[n].view(torch.int16) if out[n].dtype == torch.bfloat16 else out[n]
            for n in ("qi", "ki", "vi", "qs", "ks", "vs", "anchors")}


def run_gelu(device):
    from h3_speedkit.ops.gemm import int8_linear
    a, w, xs, ws = codes(21, 77, 256), codes(22, 256, 256), between(23, 0.005, 0.05, 77), between(24, 0.0005, 0.005, 256)
    return {"out": int8_linear(a.to(device), w.to(device), xs.to(device), ws.to(device), gelu=True).view(torch.int16)}


def outputs(device):
    """Every golden case's outputs by file name."""
    named = {f"block_attention_{n}": run_attention(n, device) for n in ATTENTION}
    named |= {f"block_qkv_{n}": run_qkv(n, device) for n in QKV}
    named["block_gelu"] = run_gelu(device)
    return {name: {k: t.cpu().numpy() for k, t in out.items()} for name, out in named.items()}
