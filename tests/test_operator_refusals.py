"""What the norm-quantiser, the rotary positions and the masked attention refuse, before
any CUDA call."""
import ctypes as ct
from types import SimpleNamespace

import pytest
import torch

from h3_speedkit import _lib
from h3_speedkit.ops import masked_attention as ma
from h3_speedkit.ops import rms_quant, rope

INVALID = 1   # cudaErrorInvalidValue
BF = torch.bfloat16


def x(m=4, k=32, t=BF):
    return torch.zeros((m, k), dtype=t)


RMS = [
    (dict(x=x(t=torch.float32)), "BF16 or FP16"),
    (dict(x=torch.zeros(4, dtype=BF)), "BF16 or FP16"),
    (dict(x=x(2, 16385), weight=torch.zeros(16385, dtype=BF)), "16384"),
    (dict(x=x(4, 0), weight=torch.zeros(0, dtype=BF)), "1 <= K"),
    (dict(x=x(4, 64)[:, ::2]), "unit columns"),
    (dict(x=x(1).expand(4, 32)), "rows apart"),
    (dict(weight=torch.zeros(31, dtype=BF)), "weight"),
    (dict(weight=torch.zeros(32, dtype=torch.float16)), "weight"),
    (dict(dtype=torch.uint8), "dtype"),
    (dict(eps=0.0), "Epsilon"),
    (dict(eps=float("nan")), "Epsilon"),
    (dict(residual_out=x()), "needs a residual"),
    (dict(residual=x(5)), "residual"),
    (dict(residual=x(), residual_out=x(1).expand(4, 32)), "residual_out"),
    (dict(residual=x(), out=torch.zeros((4, 32), dtype=torch.uint8)), "out"),
    (dict(out_scale=torch.zeros(4)), "out_scale"),
    (dict(weight=torch.zeros(32, dtype=BF, requires_grad=True)), "Inference only"),
]


@pytest.mark.parametrize("change,text", RMS)
def test_rms_quant_refuses(change, text):
    args = dict(x=x(), weight=torch.ones(32, dtype=BF)) | change
    with pytest.raises(ValueError, match=text):
        rms_quant.residual_rms_quant(args.pop("x"), args.pop("weight"), **args)


def test_rms_quant_refuses_overlaps_and_the_cpu():
    buf, w = x(8), torch.ones(32, dtype=BF)
    with pytest.raises(ValueError, match="overlaps input"):
        rms_quant.residual_rms_quant(buf[:4], w, residual=x(), residual_out=buf[2:6])
    with pytest.raises(ValueError, match="overlaps input x"):
        rms_quant.residual_rms_quant(buf[:4], w, out=buf[:2].view(torch.int8).view(4, 32))
    with pytest.raises(ValueError, match="CUDA device"):
        rms_quant.residual_rms_quant(buf[:4], w, residual=buf[4:], residual_out=buf[4:])


def run_rms(**change):
    a = dict(x=16, r=16, w=16, h=16, q=16, s=16, m=4, k=64, xs=64, rs=64, hs=64, eps=1e-6, t=0, wt=0, c=0) | change
    return _lib.load().h3_rms_quant_run(a["x"], a["r"], a["w"], a["h"], a["q"], a["s"], a["m"], a["k"], a["xs"], a["rs"],
                                        a["hs"], ct.c_float(a["eps"]), a["t"], a["wt"], a["c"], 0)


@pytest.mark.parametrize("bad", [dict(x=None), dict(w=None), dict(q=None), dict(s=None), dict(h=None), dict(m=-1), dict(m=2**31),
                                 dict(k=0), dict(k=16385), dict(xs=63), dict(rs=63), dict(hs=63), dict(eps=0.0),
                                 dict(eps=float("inf")), dict(t=2, wt=2), dict(wt=1), dict(c=2), dict(x=17), dict(s=18)])
def test_rms_entry_point_refuses(bad):
    assert run_rms(**bad) == INVALID


def test_entry_points_take_nothing_for_nothing():
    assert run_rms(m=0, x=None) == 0
    lib, turns, axis = _lib.load(), (ct.c_double * 4)(), (ct.c_int * 4)()
    assert lib.h3_rope_table_run(None, turns, axis, None, 0, 4, 1, 0, 0) == 0


def heads(t=4, h=2, d=64, dtype=BF):
    return torch.zeros((t, h, d), dtype=dtype)


def at(t=4, a=3, dtype=torch.int32):
    return torch.zeros((t, a), dtype=dtype)


ROPE = [
    (dict(positions=at(a=2)), "positions"),
    (dict(positions=at(dtype=torch.int64)), "positions"),
    (dict(positions=at(5)), "every token"),
    (dict(positions=at(4, 6)[:, ::2]), "positions"),
    (dict(sections=(8, 8, -1)), "whole numbers"),
    (dict(sections=(8, 8, 2.0)), "whole numbers"),
    (dict(sections=(0, 0, 0)), "sum"),
    (dict(sections=(64, 64, 1)), "sum"),
    (dict(sections=(2**62, 2**62, 2**62)), "sum"),
    (dict(sections=(16, 16, 1)), "hold the 33 pairs"),
    (dict(theta=0.0), "theta"),
    (dict(theta=(1e4, 1e4)), "theta"),
    (dict(theta=float("inf")), "theta"),
    (dict(q=heads(dtype=torch.float32)), "BF16 or FP16"),
    (dict(q=heads(d=63)), "even"),
    (dict(q=heads(d=258)), "even"),
    (dict(k=heads(t=3)), "k requires"),
    (dict(k=heads(dtype=torch.float16)), "k requires"),
    (dict(q=heads(d=128)[..., ::2]), "unit channels"),
    (dict(eps=0.0), "Epsilon"),
    (dict(k=None, k_out=heads()), "need k"),
    (dict(q_weight=torch.ones(64, dtype=BF)), "together"),
    (dict(q_weight=torch.ones(64, dtype=BF), k_weight=torch.ones(64)), "alike"),
    (dict(q_out=heads(h=1).expand(4, 2, 64)), "overlapping itself"),
    (dict(q_out=heads(h=3)), "q_out"),
    (dict(q=heads().requires_grad_()), "Inference only"),
]


@pytest.mark.parametrize("change,text", ROPE)
def test_rope_refuses(change, text):
    args = dict(q=heads(), k=heads(), positions=at(), sections=(8, 8, 8)) | change
    with pytest.raises(ValueError, match=text):
        rope.rope_axes(args.pop("q"), args.pop("k"), args.pop("positions"), **args)


def test_rope_outputs_in_place_or_apart():
    qkv = torch.zeros((4, 6 * 64), dtype=BF)
    q, k, v = (qkv[:, 128 * i:128 * i + 128].view(4, 2, 64) for i in range(3))
    go = dict(positions=at(), sections=(8, 8, 8))
    for out in (dict(q_out=q, k_out=k), dict(q_out=v), dict(k_out=v)):
        with pytest.raises(ValueError, match="CUDA device"):     # accepted up to the device
            rope.rope_axes(q, k, **go, **out)
    for out in (dict(q_out=k), dict(k_out=q), dict(q_out=v, k_out=v),
                dict(q_out=qkv[:, 64:192].view(4, 2, 64)), dict(q_out=qkv.view(-1)[128:128 + 512].view(4, 2, 64))):
        with pytest.raises(ValueError, match="overlap"):
            rope.rope_axes(q, k, **go, **out)


@pytest.mark.parametrize("change,text", [(dict(sections=(48, 1)), "positions"), (dict(out=torch.zeros((1, 4, 1, 24, 2, 2))), "out")])
def test_table_refuses(change, text):
    args = dict(positions=at(), sections=(8, 8, 8)) | change
    with pytest.raises(ValueError, match=text):
        rope.rope_table(args.pop("positions"), **args)


class RopeArgs(ct.Structure):
    """The C argument block H3RopeArgs (include/h3sk_b200.h)."""
    _fields_ = ([(n, ct.c_void_p) for n in ("q", "k", "q_out", "k_out", "q_weight", "k_weight", "positions", "turns", "axis")]
                + [("tokens", ct.c_int64), ("strides", ct.c_int64 * 8)]
                + [(n, ct.c_int32) for n in ("q_heads", "k_heads", "dim", "pairs", "axes", "float_positions", "type",
                                             "weight_type", "interleaved", "inverse")] + [("eps", ct.c_float)])


def rope_args(**change):
    turns, axis = (ct.c_double * 24)(), (ct.c_int * 24)(*change.pop("axis_values", [0] * 24))
    a = dict(q=16, k=16, q_out=16, k_out=16, positions=16, turns=ct.addressof(turns), axis=ct.addressof(axis), tokens=4,
             q_heads=2, k_heads=2, dim=64, pairs=24, axes=1, eps=1e-6) | change
    return _lib.load().h3_rope_axes_run(ct.byref(RopeArgs(**a)), 0)


def test_rope_struct_sizes_agree():
    assert _lib.load().h3_rope_args_size() == ct.sizeof(RopeArgs)


@pytest.mark.parametrize("bad", [dict(q=None), dict(k_out=None), dict(tokens=-1), dict(q_heads=-1), dict(q_heads=65536),
                                 dict(dim=63), dict(dim=258), dict(pairs=33), dict(pairs=0), dict(axes=0), dict(type=2, weight_type=2),
                                 dict(weight_type=1), dict(eps=0.0), dict(positions=None), dict(positions=18), dict(q=17),
                                 dict(q_weight=16), dict(turns=None), dict(axis_values=[1] * 24), dict(tokens=2**40)])
def test_rope_entry_point_refuses(bad):
    assert rope_args(**bad) == INVALID


def qkv(b=2, sq=5, sk=7, hq=4, hk=2, d=64, dtype=BF):
    return dict(q=torch.zeros((b, sq, hq, d), dtype=dtype), k=torch.zeros((b, sk, hk, d), dtype=dtype),
                v=torch.zeros((b, sk, hk, d), dtype=dtype))


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


ATTENTION = [
    (dict(q=torch.zeros((2, 5, 4, 64))), "BF16 or FP16"),
    (dict(k=torch.zeros((2, 7, 2, 64), dtype=torch.float16)), "all alike"),
    (dict(v=torch.zeros((7, 2, 64), dtype=BF)), "all alike"),
    (dict(v=torch.zeros((2, 8, 2, 64), dtype=BF)), "one shape"),
    (qkv(d=96), "D 64 or 128"),
    (qkv(hq=3), "multiple of Hk"),
    (qkv(hk=0), "multiple of Hk"),
    (dict(q=torch.zeros((2, 5, 4, 128), dtype=BF)[..., ::2]), "unit channels"),
    (dict(q=torch.zeros((2, 5, 4, 68), dtype=BF)[..., :64]), "multiples of 8"),
    (dict(k=torch.zeros(2 * 7 * 2 * 64 + 1, dtype=BF)[1:].view(2, 7, 2, 64)), "16-byte"),
    (dict(q=torch.zeros((2, 1, 4, 64), dtype=BF).expand(2, 5, 4, 64)), "expanded"),
    (dict(k=torch.zeros((2, 1, 2, 64), dtype=BF).expand(2, 7, 2, 64)), "expanded"),
    (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"),
    (dict(softcap=-1.0), "softcap"),
    (dict(softcap=float("inf")), "softcap"),
    (dict(softcap=3e38), "softcap"),
    (dict(softcap=2e-38, scale=5.0), "ratio"),
    (dict(q_offsets=i32(0, 5)), "together"),
    (dict(q_offsets=i32(0, 5), k_offsets=i32(0, 7)), "one sequence"),
    (qkv(b=1) | dict(q_offsets=i32(0), k_offsets=i32(0)), "at least one document"),
    (qkv(b=1) | dict(q_offsets=i32(0, 5), k_offsets=i32(0, 5, 7)), "k_offsets requires"),
    (qkv(b=1) | dict(q_offsets=i32(0, 5).long(), k_offsets=i32(0, 7)), "q_offsets requires"),
    (qkv(b=1) | dict(q_offsets=i32(0, 5), k_offsets=i32(0, 7), k_lengths=i32(7)), "without lengths"),
    (dict(q_lengths=i32(5)), "q_lengths requires"),
    (dict(k_lengths=i32(5, 5, 5)), "k_lengths requires"),
    (dict(prefix=i32(1, 1)), "causal=True"),
    (dict(prefix=i32(1), causal=True), "prefix requires"),
    (dict(slopes=torch.zeros(2)), "slopes"),
    (dict(slopes=torch.zeros(4, dtype=BF)), "slopes"),
    (dict(out=torch.zeros((2, 5, 4, 64))), "out requires"),
    (dict(out=torch.zeros((2, 5, 1, 64), dtype=BF).expand(2, 5, 4, 64)), "overlap itself"),
    (dict(lse=torch.zeros((2, 5, 4))), "lse requires"),
    (dict(q=torch.zeros((2, 5, 4, 64), dtype=BF, requires_grad=True)), "Inference only"),
    (dict(), "CUDA device"),
]


@pytest.mark.parametrize("change,text", ATTENTION)
def test_masked_attention_refuses(change, text):
    args = qkv() | change
    with pytest.raises(ValueError, match=text):
        ma.masked_attention(args.pop("q"), args.pop("k"), args.pop("v"), **args)


def test_masked_attention_refuses_overlaps():
    args = qkv()
    with pytest.raises(ValueError, match="overlaps q"):
        ma.masked_attention(**args, out=args["q"])
    both = torch.zeros(2 * 5 * 4 * 64 * 2, dtype=BF)
    with pytest.raises(ValueError, match="overlaps"):
        ma.masked_attention(**args, out=both[:2560].view(2, 5, 4, 64), lse=both.view(torch.float32)[:40].view(2, 4, 5))


def test_provider_refuses():
    with pytest.raises(ValueError, match="together"):
        ma.MaskedAttentionProvider(4, positions=at())
    with pytest.raises(ValueError, match="divide"):
        ma.MaskedAttentionProvider(3)(*(torch.zeros((4, 128), dtype=BF) for _ in range(3)))


class AttentionArgs(ct.Structure):
    """The C argument block H3MaskedAttentionArgs (include/h3sk_b200.h)."""
    _fields_ = ([(n, ct.c_void_p) for n in ("q", "k", "v", "out", "lse", "slopes", "q_offsets", "k_offsets", "q_lengths",
                                            "k_lengths", "prefix", "workspace")] + [("workspace_bytes", ct.c_uint64)]
                + [(f"{t}_stride_{d}", ct.c_int64) for t in "qkvo" for d in "bsh"]
                + [(n, ct.c_int32) for n in ("batch", "q_len", "k_len", "q_heads", "k_heads", "dim", "type", "documents", "causal",
                                             "fill")]
                + [("scale", ct.c_float), ("softcap", ct.c_float)])


def attention_args(**change):
    a = dict(q=16, k=16, v=16, out=16, batch=2, q_len=5, k_len=7, q_heads=4, k_heads=2, dim=64, scale=0.125,
             q_stride_b=1280, q_stride_s=256, q_stride_h=64, k_stride_b=896, k_stride_s=128, k_stride_h=64, v_stride_b=896,
             v_stride_s=128, v_stride_h=64, o_stride_b=1280, o_stride_s=256, o_stride_h=64) | change
    return _lib.load().h3_masked_attention_run(ct.byref(AttentionArgs(**a)), 0)


@pytest.mark.parametrize("bad", [dict(q=None), dict(out=None), dict(k=None), dict(v=None), dict(batch=-1), dict(q_len=-1),
                                 dict(k_len=-1), dict(q_len=2**30 + 1), dict(q_heads=3), dict(k_heads=0), dict(dim=96), dict(type=2),
                                 dict(documents=-1), dict(documents=1), dict(q_offsets=16, k_offsets=16), dict(prefix=16),
                                 dict(scale=0.0), dict(scale=float("inf")), dict(softcap=-1.0), dict(softcap=1e-38, scale=9.0),
                                 dict(q_stride_s=255),
                                 dict(v_stride_h=-64), dict(o_stride_s=0), dict(q_stride_h=0), dict(k_stride_s=0), dict(q=24),
                                 dict(out=8), dict(lse=18), dict(k_lengths=18)])
def test_masked_attention_entry_point_refuses(bad):
    assert attention_args(**bad) == INVALID


def test_masked_attention_struct_and_nothing_to_do():
    lib = _lib.load()
    assert lib.h3_masked_attention_args_size() == ct.sizeof(AttentionArgs)
    assert lib.h3_masked_attention_run(None, 0) == INVALID and lib.h3_masked_attention_workspace(None) == -1
    assert lib.h3_masked_attention_plan(None, (ct.c_int * 3)()) == INVALID
    assert attention_args(batch=0, q=None) == 0 and attention_args(q_len=0, out=None) == 0


class Subclass(torch.Tensor):
    pass


def kinds(t):
    """A tensor as no operator of this package takes it: a subclass, a Parameter, one that is
    negated on reading, one without memory."""
    yield t.as_subclass(Subclass), "original plain"
    yield torch.nn.Parameter(t, requires_grad=False), "original plain"
    yield torch._neg_view(t), "original plain"
    yield torch._efficientzerotensor(t.shape, dtype=t.dtype), "original plain"
    yield t.clone().requires_grad_(), "Inference only"


CALLS = {  # operator, operands by name
    "rms_quant": (rms_quant.residual_rms_quant, lambda: dict(
        x=x(), weight=torch.ones(32, dtype=BF), residual=x(), residual_out=x())),
    "rope_axes": (rope.rope_axes, lambda: dict(
        q=heads(), k=heads(), positions=at(dtype=torch.float32), sections=(8, 8, 8), q_weight=torch.ones(64),
        k_weight=torch.ones(64), q_out=heads(), k_out=heads())),
    "rope_table": (rope.rope_table, lambda: dict(
        positions=at(dtype=torch.float32), sections=(8, 8, 8), out=torch.zeros((1, 4, 1, 24, 2, 2), dtype=BF))),
    "masked_attention": (ma.masked_attention, lambda: qkv() | dict(
        slopes=torch.zeros(4), out=torch.zeros((2, 5, 4, 64), dtype=BF), lse=torch.zeros((2, 4, 5)))),
}


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", list(CALLS))
def test_operands_are_plain_tensors_without_a_gradient(name, grad):
    """Whether gradients are recorded at the time or not, as in the package's other operators."""
    import torch.autograd.forward_ad as forward
    call, operands = CALLS[name]
    for key, t in operands().items():
        if not isinstance(t, torch.Tensor):
            continue
        for other, text in kinds(t):
            with torch.set_grad_enabled(grad), pytest.raises(ValueError, match=text):
                call(**operands() | {key: other})
        with forward.dual_level(), pytest.raises(ValueError, match="Inference only"):
            call(**operands() | {key: forward.make_dual(t, torch.ones_like(t))})
    with pytest.raises(ValueError, match="CUDA device"):     # and nothing else is wrong
        call(**operands())


@pytest.mark.parametrize("q_type,k_type,want", [(BF, BF, BF), (torch.float32, torch.float32, torch.float32),
                                                (BF, torch.float32, torch.float32), (torch.float16, torch.float16, torch.float32)])
def test_provider_keeps_the_norm_weights_digits(monkeypatch, q_type, k_type, want):
    """Norm weights reach the rotation as they are stored: a BF16 Q does not round FP32 ones."""
    weights = [(1 + 0.1 * torch.arange(128) / 128).to(t) for t in (q_type, k_type)]
    block = SimpleNamespace(attn=SimpleNamespace(**{n: SimpleNamespace(weight=torch.nn.Parameter(w), eps=1e-6)
                                                    for n, w in zip(("q_norm", "k_norm"), weights)}))
    seen = {}
    monkeypatch.setattr(ma, "rope_axes", lambda q, k, at, **more: seen.update(more) or (q, k))
    monkeypatch.setattr(ma, "masked_attention", lambda q, k, v, **masks: v)
    provider = ma.MaskedAttentionProvider(2, positions=at(), sections=(16, 16, 16))
    provider.for_block(block)(*(torch.zeros((4, 256), dtype=BF) for _ in range(3)))
    for name, w in zip(("q_weight", "k_weight"), weights):
        assert seen[name].dtype == want and torch.equal(seen[name].double(), w.double())


def test_provider_takes_masks_alone():
    """The block wants the attention's result and nothing else: no outputs of the caller's, no lse."""
    for other in (dict(return_lse=True), dict(out=torch.zeros((4, 2, 64), dtype=BF)), dict(lse=torch.zeros((2, 4))), dict(mask=None)):
        with pytest.raises(ValueError, match="masks are any of"):
            ma.MaskedAttentionProvider(2, causal=True, **other)
    assert ma.MaskedAttentionProvider(2, causal=True, softcap=3.0).masks == dict(causal=True, softcap=3.0)
