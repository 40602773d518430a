"""masked_attention against the definition in 64 bits."""
import ctypes as ct
import math
from types import SimpleNamespace

import pytest
import torch

from h3_speedkit import _lib
from h3_speedkit.ops.masked_attention import MaskedAttentionProvider, masked_attention

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def definition(q, k, v, spans, *, scale, cap=0.0, slopes=None, causal=False, prefix=None):
    """(out, lse, error bound of out, of lse); spans: (batch, q0, q1, k0, k1) of each sequence.

    The bound: probabilities are rounded to the type (half a step each of sum p|v|), the
    result once more; a score is off by its FP32 sum of D products, taken as 4e-6 of the
    largest score before the cap and of the cap, and moves a weight by that much."""
    b, sq, hq, d = q.shape
    g = hq // k.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.zeros((b, hq, sq), dtype=torch.float64, device=q.device)
    out_err, lse_err, half = torch.zeros_like(out), torch.zeros_like(lse), torch.finfo(q.dtype).eps / 2
    for n, (bi, q0, q1, k0, k1) in enumerate(spans):
        if q1 == q0:
            continue
        pos = torch.arange(q1 - q0, device=q.device)[:, None] + (k1 - k0) - (q1 - q0)
        j = torch.arange(k1 - k0, device=q.device)[None]
        see = torch.ones((q1 - q0, k1 - k0), dtype=torch.bool, device=q.device)
        if causal:
            see = (j <= pos) | (j < (int(prefix[n]) if prefix is not None else 0))
        for h in range(hq):
            s = q[bi, q0:q1, h].double() @ k[bi, k0:k1, h // g].double().T * scale
            raw = s.masked_fill(~see, 0).abs().amax(1, keepdim=True) if s.shape[1] else s.new_zeros((q1 - q0, 1))
            if cap:
                s = cap * torch.tanh(s / cap)
            if slopes is not None:
                s = s - slopes[h].double() * (pos - j).abs()
            s = s.masked_fill(~see, -INF)
            total = torch.logsumexp(s, 1, keepdim=True) if s.shape[1] else s.new_full((q1 - q0, 1), -INF)
            w = torch.where(see & (total > -INF), torch.exp(s - total), 0.0)
            val = v[bi, k0:k1, h // g].double()
            out[bi, q0:q1, h] = w @ val
            lse[bi, h, q0:q1] = total[:, 0]
            err = 4e-6 * (1 + raw + cap)
            # + what FP16 loses below its subnormals (probabilities are scaled by 2^7)
            lost = val.abs().amax(0) * (k1 - k0) * 2.0 ** -32 if len(val) else 0.0
            out_err[bi, q0:q1, h] = (half * 1.01 + 2 * err) * (w @ val.abs()) + half * 1.01 * out[bi, q0:q1, h].abs() + lost + 1e-7
            lse_err[bi, h, q0:q1] = err[:, 0] + 1e-6 * (1 + lse[bi, h, q0:q1].abs().nan_to_num(posinf=0.0))
    return out, lse, out_err, lse_err


def check(got, want, rows=None):
    out, lse = got
    ref, ref_lse, err, lse_err = want
    rows = slice(None) if rows is None else rows
    bad = ((out.double() - ref).abs() > err)[:, rows]
    assert not bad.any(), (int(bad.sum()), float(((out.double() - ref).abs() / err)[:, rows].max()))
    a, b = lse[..., rows].double(), ref_lse[..., rows]
    empty = torch.isinf(b)
    assert torch.equal(a[empty], b[empty])
    assert torch.all((a - b).abs()[~empty] <= lse_err[..., rows][~empty])
    assert not torch.isnan(out[:, rows]).any()


def make(b, sq, sk, hq, hk, d, t, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed + sq * 7 + sk)
    q, k, v = (torch.randn((b, s, h, d), generator=g, device=device) for s, h in ((sq, hq), (sk, hk), (sk, hk)))
    return (2 * q).to(t), k.to(t), v.to(t)


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


@pytest.fixture(autouse=True)
def no_late_waits():
    yield
    assert _lib.pipeline_status() == 0


@pytest.mark.parametrize("sq,sk", [(1, 1), (1, 127), (1, 128), (1, 129), (3, 1000), (128, 128), (127, 300), (129, 257), (256, 256),
                                   (257, 1), (300, 511), (640, 1153), (5, 0)])
@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 4), (8, 2), (7, 1), (6, 2)])
@pytest.mark.parametrize("d,t", [(128, torch.bfloat16), (64, torch.float16), (128, torch.float16), (64, torch.bfloat16)])
def test_every_key(device, sq, sk, hq, hk, d, t):
    q, k, v = make(2, sq, sk, hq, hk, d, t, device)
    got = masked_attention(q, k, v, return_lse=True)
    check(got, definition(q, k, v, [(b, 0, sq, 0, sk) for b in range(2)], scale=d ** -0.5))


@pytest.mark.parametrize("cap,distance", [(0.0, False), (20.0, False), (0.0, True), (50.0, True)])
@pytest.mark.parametrize("sq,sk,causal,prefix", [(300, 300, True, None), (300, 300, True, [40, 299]), (64, 700, True, None),
                                                 (700, 64, True, None), (700, 64, True, [10, 0]), (1, 1000, True, None),
                                                 (333, 200, False, None), (130, 1030, True, [1030, 2000])])
def test_causal_prefix_cap_and_distance(device, sq, sk, causal, prefix, cap, distance):
    """700 queries over 64 keys leave the first rows without a key."""
    for d, t in ((128, torch.bfloat16), (64, torch.float16)):
        q, k, v = make(2, sq, sk, 6, 3, d, t, device)
        slopes = torch.exp2(-torch.arange(1, 7, device=device).float()) if distance else None
        got = masked_attention(q, k, v, causal=causal, prefix=None if prefix is None else ints(prefix, device), softcap=cap,
                               slopes=slopes, return_lse=True)
        check(got, definition(q, k, v, [(b, 0, sq, 0, sk) for b in range(2)], scale=d ** -0.5, cap=cap, slopes=slopes,
                              causal=causal, prefix=prefix))


@pytest.mark.parametrize("lengths", [[0, 1, 2, 130, 0, 0, 255, 64, 700, 1], [1] * 300, [513], [0, 0, 7], [300, 0, 900, 5, 128, 256]])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk", [(4, 4), (8, 1)])
def test_documents(device, lengths, causal, hq, hk):
    """Packed documents, keys of other lengths than the queries; rows before the first and
    behind the last document stay."""
    t, d = torch.bfloat16, 128
    klens = [n + (3 * i) % 5 if n else (0 if i % 2 else 4) for i, n in enumerate(lengths)]
    qo = [5 + sum(lengths[:i]) for i in range(len(lengths) + 1)]
    ko = [2 + sum(klens[:i]) for i in range(len(lengths) + 1)]
    q, k, v = make(1, qo[-1] + 9, ko[-1] + 3, hq, hk, d, t, device)
    prefix = [(7 * i) % 13 for i in range(len(lengths))]
    args = dict(q_offsets=ints(qo, device), k_offsets=ints(ko, device), causal=causal,
                prefix=ints(prefix, device) if causal else None)
    spans = [(0, qo[i], qo[i + 1], ko[i], ko[i + 1]) for i in range(len(lengths))]
    want = definition(q, k, v, spans, scale=d ** -0.5, causal=causal, prefix=prefix)
    out, lse = torch.full_like(q, 7.0), torch.full((1, hq, q.shape[1]), 7.0, device=device)
    got = masked_attention(q, k, v, out=out, lse=lse, **args)
    inside = slice(qo[0], qo[-1])
    check(got, want, inside)
    for rows in (slice(0, qo[0]), slice(qo[-1], None)):
        assert torch.all(out[:, rows] == 7.0) and torch.all(lse[..., rows] == 7.0)
    fresh = masked_attention(q[0], k[0], v[0], return_lse=True, **args)    # one sequence in three dimensions
    assert torch.equal(fresh[0][inside], out[0, inside]) and torch.equal(fresh[1][:, inside], lse[0][:, inside])
    assert torch.all(fresh[0][:qo[0]] == 0) and torch.all(fresh[1][:, qo[-1]:] == 0)


@pytest.mark.parametrize("sq,qlens,klens", [(333, [333, 0, 128, 1], [333, 0, 128, 1]), (1, None, [1000, 0, 1, 513]),
                                            (200, [200, 199, 1, 0], None), (40, [40, 3, 0, 7], [1000, 2, 5, 0])])
def test_padded_batch_and_values_behind_the_sequences(device, sq, qlens, klens):
    """NaN and infinities behind the valid tokens reach nothing."""
    b, sk, d, t = 4, sq if sq == 333 else 1000, 128, torch.bfloat16
    q, k, v = make(b, sq, sk, 4, 2, d, t, device)
    kn, qn = klens or [sk] * b, qlens or [sq] * b
    for i in range(b):
        k[i, kn[i]:], v[i, kn[i]:], q[i, qn[i]:] = NAN, (NAN, INF, 3e38, -3e38)[i], NAN
    want = definition(q, k, v, [(i, 0, qn[i], 0, kn[i]) for i in range(b)], scale=d ** -0.5)
    out, lse = masked_attention(q, k, v, q_lengths=None if qlens is None else ints(qlens, device),
                                k_lengths=None if klens is None else ints(klens, device), return_lse=True)
    for i in range(b):
        one = tuple(x[i:i + 1] for x in want)
        check((out[i:i + 1], lse[i:i + 1]), one, slice(0, qn[i]))
        assert qlens is None or torch.all(out[i, qn[i]:] == 0)


@pytest.mark.parametrize("pair", [True, False])
def test_not_finite_values_reach_those_who_see_them(device, pair):
    """A document with NaN in V, one with an infinity, neighbours in the same key block."""
    lens = [100, 60, 70, 90] * (20 if pair else 1)
    offs = [sum(lens[:i]) for i in range(len(lens) + 1)]
    q, k, v = make(1, offs[-1], offs[-1], 4 if not pair else 40, 4 if not pair else 40, 128, torch.bfloat16, device)
    clean = masked_attention(q, k, v, q_offsets=ints(offs, device), k_offsets=ints(offs, device))
    v[0, offs[1] + 3, 1, 17] = NAN
    v[0, offs[2] + 5, 2, 90] = -INF
    k[0, offs[1] + 9, 0, 3] = NAN
    out = masked_attention(q, k, v, q_offsets=ints(offs, device), k_offsets=ints(offs, device))
    want = clean.clone()
    want[0, offs[1]:offs[2], 1, 17] = NAN
    want[0, offs[2]:offs[3], 2, 90] = -INF
    want[0, offs[1]:offs[2], 0] = NAN
    assert torch.equal(torch.nan_to_num(out, 5.0), torch.nan_to_num(want, 5.0))
    assert torch.equal(torch.isnan(out), torch.isnan(want))


def test_large_and_growing_scores(device):
    """The row maximum grows by far more than 2^8 again and again, or falls."""
    d, t = 128, torch.float16
    q, k, v = make(1, 200, 1500, 2, 2, d, t, device)
    ramp = torch.linspace(0.0, 8.0, 1500, device=device)
    q[..., 0] = 8.0
    for sign in (1.0, -1.0):
        k[..., 0] = (sign * ramp * 8).to(t)[None, :, None]
        got = masked_attention(q, k, v, scale=1.0, return_lse=True)
        check(got, definition(q, k, v, [(0, 0, 200, 0, 1500)], scale=1.0))


def test_scores_of_minus_infinity_and_overflow(device):
    q, k, v = make(1, 4, 300, 1, 1, 64, torch.bfloat16, device)
    q[..., 0], k[..., 0] = 1.0, -INF
    out, lse = masked_attention(q, k, v, return_lse=True)
    assert torch.all(out == 0) and torch.all(lse == -INF)       # nothing to weigh: as an empty row
    k[:, 7, :, 0] = 0.0
    out, lse = masked_attention(q, k, v, return_lse=True)
    assert torch.equal(out[0, :, 0], v[0, 7].expand(4, 64)) and torch.isfinite(lse).all()
    k[:, 9, :, 0] = INF
    assert torch.isnan(masked_attention(q, k, v)).all()


@pytest.mark.parametrize("form", ["projection", "expanded", "heads first", "padded rows"])
def test_strides(device, form):
    d, t = 128, torch.bfloat16
    if form == "projection":
        qkv = torch.randn((300, 12 * d), device=device).to(t)
        q, k, v = (qkv[None, :, a * d:b * d].view(1, 300, -1, d) for a, b in ((0, 8), (8, 10), (10, 12)))
    elif form == "expanded":
        q, k, v = make(3, 100, 200, 4, 4, d, t, device)
        q, k, v = q[:1].expand(3, 100, 4, d), k[:1, :, :1].expand(3, 200, 4, d), v[:, :, :1].expand(3, 200, 4, d)
    elif form == "heads first":
        q, k, v = (torch.randn((2, 4, n, d), device=device).to(t).transpose(1, 2) for n in (150, 260, 260))
    else:
        q, k, v = (torch.randn((2, n, 4, d + 8), device=device).to(t)[..., 8:] for n in (150, 260, 260))
    out = torch.empty((*q.shape[:3], 2 * d), device=device, dtype=t)[..., d:] if form == "padded rows" else None
    got = masked_attention(q, k, v, out=out, return_lse=True)
    assert out is None or got[0] is out
    check(got, definition(q, k, v, [(b, 0, q.shape[1], 0, k.shape[1]) for b in range(q.shape[0])], scale=d ** -0.5))


@pytest.mark.parametrize("hq,hk,sq,b", [(56, 8, 1, 2), (3, 3, 2, 1), (16, 1, 9, 1), (2, 2, 130, 1)])
def test_split_keys(device, hq, hk, sq, b):
    """Few rows over long keys: the keys are split over CTAs and joined."""
    lib_args = make(b, sq, 20000, hq, hk, 128, torch.bfloat16, device)
    got = masked_attention(*lib_args, return_lse=True, causal=True)
    check(got, definition(*lib_args, [(i, 0, sq, 0, 20000) for i in range(b)], scale=128 ** -0.5, causal=True))


def test_more_than_2_31_values(device):
    """Offsets into a long cache pass 32 bits: the last sequence's keys lie behind 2^31 values."""
    b, sk, hk, d = 18, 131072, 8, 128
    cache = torch.zeros((b, sk, 2, hk, d), dtype=torch.bfloat16, device=device)
    q, k, v = make(1, 3, 300, 8, hk, d, torch.bfloat16, device)
    cache[-1, -300:, 0], cache[-1, -300:, 1] = k[0], v[0]
    o = ints([0, 3], device), ints([sk - 300, sk], device)
    got = masked_attention(q, cache[-1:, :, 0], cache[-1:, :, 1], q_offsets=o[0], k_offsets=o[1], return_lse=True)
    want = masked_attention(q, k, v, return_lse=True)
    assert cache.numel() > 2 ** 31
    assert torch.allclose(got[0].float(), want[0].float(), rtol=2 ** -7, atol=2 ** -8)
    all_keys = masked_attention(q.expand(b, 3, 8, d), cache[:, :, 0], cache[:, :, 1], k_lengths=ints([sk] * b, device))
    last = masked_attention(q, cache[-1:, :, 0], cache[-1:, :, 1])
    assert torch.allclose(all_keys[-1:].float(), last.float(), rtol=2 ** -7, atol=2 ** -10)


def test_same_bits_on_streams_and_in_graphs(device):
    q, k, v = make(1, 17, 9000, 8, 2, 128, torch.bfloat16, device)
    lengths = ints([9000], device)
    want = masked_attention(q, k, v, k_lengths=lengths, return_lse=True)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:                              # two calls at once, each with its own workspace
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([masked_attention(q, k, v, k_lengths=lengths, return_lse=True) for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for g in got for one in g for x, y in zip(one, want))
    graphs, held, state = [], [], (q.clone(), lengths.clone())
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(masked_attention(state[0], k, v, k_lengths=state[1], return_lse=True))
        graphs.append(graph)
    state[0].copy_(q.flip(1))
    state[1].fill_(4321)
    for s, graph in zip(streams, graphs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    again = masked_attention(q.flip(1), k, v, k_lengths=ints([4321], device), return_lse=True)
    assert all(torch.equal(x, y) for h in held for x, y in zip(h, again))


def test_block_path(device):
    """The provider behind Backend.block: norm, projection, positions, masks, out-projection,
    against the same steps called one by one."""
    from h3_speedkit.ops.gemm import int8_linear
    from h3_speedkit.ops.rms_quant import residual_rms_quant
    from h3_speedkit.ops.rope import rope_axes
    g = torch.Generator(device=device).manual_seed(5)
    m, heads, hidden = 200, 4, 512
    x, r = (torch.randn((m, hidden), generator=g, device=device).bfloat16() for _ in range(2))
    w = (1 + 0.1 * torch.rand(hidden, generator=g, device=device)).bfloat16()
    wq = torch.randint(-127, 128, (3 * heads * 128, hidden), generator=g, device=device, dtype=torch.int8)
    ws = torch.full((3 * heads * 128,), 2e-4, device=device)
    at = torch.stack([torch.arange(m, device=device) // 40, torch.arange(m, device=device) % 40 // 8,
                      torch.arange(m, device=device) % 8], 1).int()
    qw, kw = (1 + 0.1 * torch.rand((2, 128), generator=g, device=device)).bfloat16()
    offs = ints([0, 77, 200], device)
    norm = lambda weight: SimpleNamespace(weight=weight, eps=1e-6)
    block = SimpleNamespace(attn=SimpleNamespace(q_norm=norm(qw), k_norm=norm(kw)))
    provider = MaskedAttentionProvider(heads, positions=at, sections=(16, 16, 16), q_offsets=offs, k_offsets=offs)
    codes, scale, h = residual_rms_quant(x, w, residual=r)
    qkv = int8_linear(codes, wq, scale, ws)
    q, k, v = qkv.split(heads * 128, 1)
    got = provider.for_block(block)(q, k, v)
    # the same in 64 bits from the projection on
    turn = lambda t, weight: rope_axes(t.view(m, heads, 128), None, at, sections=(16, 16, 16), q_weight=weight)[0][None]
    want = definition(turn(q, qw), turn(k, kw), v.view(1, m, heads, 128), [(0, 0, 77, 0, 77), (0, 77, 200, 77, 200)],
                      scale=128 ** -0.5)
    err = (got.view(1, m, heads, 128).double() - want[0]).abs()
    assert torch.all(err <= want[2])
    # the result goes on through the norm-quantiser into the next linear
    codes2, scale2, h2 = residual_rms_quant(got, w, residual=h)
    assert torch.equal(h2, (got.float() + h.float()).bfloat16())
    out = int8_linear(codes2, wq, scale2, ws)
    # (the sum of whole numbers is exact, so a sum of zero stays zero)
    back = (codes2.double() @ wq.double().T) * scale2.double() * ws.double()
    assert torch.all((out.double() - back).abs() <= back.abs() * 2.0 ** -8 * 1.001)
    assert math.isfinite(out.float().sum().item())


def test_backend_block_takes_the_provider(device):
    """Backend.block with a provider is the block with its steps called by hand."""
    from h3_speedkit import synthetic
    from h3_speedkit.ops.rope import rope_axes
    from h3_speedkit.runtime import Backend
    from test_gpu_attention import _h3_block_ns
    m, heads = 300, 56
    bw = synthetic.h3_block(0, tables=2, device=device)
    g = torch.Generator(device=device).manual_seed(11)
    qw, kw = (torch.rand((2, 128), generator=g, device=device) + 0.5).bfloat16()
    at = torch.randint(0, 50, (m, 3), generator=g, device=device, dtype=torch.int32)
    offs = ints([0, 90, 91, m], device)
    rows = (torch.arange(m, device=device) % 2).to(torch.int32)
    x0, block = synthetic.cfg5_tokens(m, 5376, device=device), _h3_block_ns(bw, qw, kw)

    def by_hand(q, k, v):
        q, k, v = (t.view(m, heads, 128) for t in (q, k, v))
        q, k = rope_axes(q, k, at, sections=(16, 16, 16), q_weight=qw, k_weight=kw)
        return masked_attention(q, k, v, q_offsets=offs, k_offsets=offs).view(m, heads * 128)
    provider = MaskedAttentionProvider(heads, positions=at, sections=(16, 16, 16), q_offsets=offs, k_offsets=offs)
    got, want = x0.clone(), x0.clone()
    Backend().block(block, got, None, None, rows=rows, attention=provider, mlp_act="swiglu")
    Backend().block(block, want, None, None, rows=rows, attention=by_hand, mlp_act="swiglu")
    assert torch.equal(got, want) and not torch.equal(got, x0)


def test_numbers_of_rows_that_fill_no_tile(device):
    """Heads of a group share a tile: sizes around the tile's ends, and a group too large for one."""
    for hq, hk, sq in ((129, 1, 3), (128, 1, 2), (65, 1, 2), (12, 4, 43), (5, 1, 26), (2, 1, 129)):
        q, k, v = make(1, sq, 200, hq, hk, 64, torch.float16, device)
        got = masked_attention(q, k, v, return_lse=True, causal=True)
        check(got, definition(q, k, v, [(0, 0, sq, 0, 200)], scale=0.125, causal=True))


def test_many_documents(device):
    """More documents than one search step holds, of every small length."""
    lens = [i % 5 for i in range(3000)]
    offs = [sum(lens[:i]) for i in range(len(lens) + 1)]
    q, k, v = make(1, offs[-1], offs[-1], 2, 1, 64, torch.bfloat16, device)
    got = masked_attention(q, k, v, q_offsets=ints(offs, device), k_offsets=ints(offs, device), return_lse=True)
    spans = [(0, a, b, a, b) for a, b in zip(offs, offs[1:]) if b > a]
    check(got, definition(q, k, v, spans, scale=0.125))


def test_capped_scores_beyond_the_polynomial(device):
    """|score| far above the cap, and rows on both sides of it in one tile."""
    q, k, v = make(1, 150, 400, 2, 2, 128, torch.bfloat16, device)
    q[:, ::3] *= 20
    for cap in (1.0, 5.0, 50.0):
        got = masked_attention(q, k, v, softcap=cap, return_lse=True)
        check(got, definition(q, k, v, [(0, 0, 150, 0, 400)], scale=128 ** -0.5, cap=cap))


def test_huge_finite_values_behind_the_sequence(device):
    """A masked key's weight is exactly zero: 3e38 times the smallest number would show."""
    for sq, sk, n in ((1, 400, 300), (300, 400, 300), (300, 128, 70)):
        q, k, v = make(1, sq, sk, 2, 2, 128, torch.bfloat16, device)
        want = masked_attention(q, k[:, :n], v[:, :n])
        v[:, n:] = 3e38
        got = masked_attention(q, k, v, k_lengths=ints([n], device))
        assert torch.equal(got, want)


def test_rows_without_keys_beside_nothing(device):
    """Tiles whose rows see no key at all are zeros, every time (nothing is computed there)."""
    q, k, v = make(2, 3000, 64, 8, 8, 128, torch.bfloat16, device)
    for _ in range(20):
        out, lse = masked_attention(q, k, v, causal=True, return_lse=True)
        assert torch.all(out[:, :2936] == 0) and torch.all(lse[..., :2936] == -INF)
        assert torch.all(masked_attention(q, k, v, k_lengths=ints([0, 0], device)) == 0)


def test_long_run_of_empty_documents(device):
    n = 200000
    offs = torch.full((n + 2,), 100, dtype=torch.int32, device=device)
    offs[0], offs[-1] = 0, 260
    q, k, v = make(1, 260, 260, 1, 1, 64, torch.bfloat16, device)
    got = masked_attention(q, k, v, q_offsets=offs, k_offsets=offs, return_lse=True)
    check(got, definition(q, k, v, [(0, 0, 100, 0, 100), (0, 100, 260, 100, 260)], scale=0.125))


def test_join_of_rows_of_no_sequence(device):
    """Split keys where most or all rows belong to no sequence, and work right behind."""
    q, k, v = make(1, 16, 20000, 2, 2, 128, torch.bfloat16, device)
    for n in (0, 1, 16):
        out = torch.full_like(q, 3.0)
        masked_attention(q, k, v, q_lengths=ints([n], device), out=out)
        doubled = out * 2                       # runs behind the join
        assert torch.all(doubled[:, n:] == 6.0)
        new, lse = masked_attention(q, k, v, q_lengths=ints([n], device), return_lse=True)
        assert torch.equal(new[:, :n], out[:, :n]) and torch.all(new[:, n:] == 0) and torch.all(lse[..., n:] == 0)
        given = torch.full_like(lse, 5.0)       # one output given, one new
        both = masked_attention(q, k, v, q_lengths=ints([n], device), lse=given)
        assert torch.equal(both[0], new) and torch.equal(given[..., :n], lse[..., :n]) and torch.all(given[..., n:] == 5.0)
        if n:
            want = definition(q[:, :n], k, v, [(0, 0, n, 0, 20000)], scale=128 ** -0.5)
            assert torch.all((out[:, :n].double() - want[0]).abs() <= want[2])


def plan(q, k, documents=0, causal=False):
    """(by pairs, heads in a tile, splits) of a call."""
    from test_operator_refusals import AttentionArgs
    a = AttentionArgs(batch=q.shape[0], q_len=q.shape[1], k_len=k.shape[1], q_heads=q.shape[2], k_heads=k.shape[2],
                      dim=q.shape[3], scale=0.1, documents=documents, causal=int(causal))
    if documents:
        a.q_offsets = a.k_offsets = 16
    out = (ct.c_int * 3)()
    assert _lib.load().h3_masked_attention_plan(ct.byref(a), out) == 0
    return tuple(out)


@pytest.mark.parametrize("cap,distance", [(0.0, False), (30.0, False), (0.0, True), (30.0, True)])
@pytest.mark.parametrize("d,t", [(128, torch.bfloat16), (64, torch.float16)])
@pytest.mark.parametrize("hq,hk", [(74, 74), (70, 10)])
def test_pairs_of_tiles(device, cap, distance, d, t, hq, hk):
    """The form that long inputs take, with every mask; odd sizes leave the last pair half
    empty, and groups of 7 leave rows of a tile unused."""
    n = 1000
    q, k, v = make(1, n, n, hq, hk, d, t, device)
    slopes = torch.exp2(-0.1 * torch.arange(1, hq + 1, device=device)) if distance else None
    more = dict(softcap=cap, slopes=slopes, return_lse=True)
    ref = dict(scale=d ** -0.5, cap=cap, slopes=slopes)
    assert plan(q, k) == (1, hq // hk, 1)
    check(masked_attention(q, k, v, **more), definition(q, k, v, [(0, 0, n, 0, n)], **ref))
    assert plan(q, k, causal=True)[0] == 1
    check(masked_attention(q, k, v, causal=True, prefix=ints([333], device), **more),
          definition(q, k, v, [(0, 0, n, 0, n)], causal=True, prefix=[333], **ref))
    lens = [100, 0, 1, 300, 90, n - 491]
    offs = [sum(lens[:i]) for i in range(len(lens) + 1)]
    assert plan(q, k, documents=len(lens))[0] == 1
    check(masked_attention(q, k, v, q_offsets=ints(offs, device), k_offsets=ints(offs, device), **more),
          definition(q, k, v, [(0, a, b, a, b) for a, b in zip(offs, offs[1:])], **ref))
    k[:, 777:], v[:, 777:] = NAN, INF
    check(masked_attention(q, k, v, k_lengths=ints([777], device), **more),
          definition(q, k, v, [(0, 0, n, 0, 777)], **ref))


def test_forms_of_the_other_tests(device):
    """Single tiles, split keys (also of pairs) and grouped heads are what the smaller tests run."""
    for sq, sk, hq, hk, want in ((300, 511, 4, 4, (0, 1, 1)), (300, 511, 8, 2, (0, 4, 1)), (1, 20000, 56, 8, (0, 7, 37)),
                                 (130, 20000, 2, 2, (0, 1, 74)), (256, 20000, 8, 8, (1, 1, 18))):
        q, k, _ = make(1, sq, sk, hq, hk, 128, torch.bfloat16, device)
        assert plan(q, k) == want


@pytest.mark.parametrize("d,t,causal,cap", [(128, torch.bfloat16, False, 0.0), (64, torch.float16, True, 30.0)])
def test_split_pairs_of_tiles(device, d, t, causal, cap):
    q, k, v = make(1, 250, 20000, 8, 8, d, t, device)
    assert plan(q, k, causal=causal)[0] == 1 and plan(q, k, causal=causal)[2] > 8
    got = masked_attention(q, k, v, causal=causal, softcap=cap, return_lse=True)
    check(got, definition(q, k, v, [(0, 0, 250, 0, 20000)], scale=d ** -0.5, causal=causal, cap=cap))


@pytest.mark.parametrize("rows,keys", [(1, 513), (1, 1100), (1, 2300), (3, 40000), (127, 3000), (250, 5000)])
@pytest.mark.parametrize("d", [64, 128])
def test_few_and_many_splits(device, rows, keys, d):
    """Keys from 128 a CTA, joined by a warp or by a CTA a row; two sequences, the second padded."""
    q, k, v = make(2, rows, keys, 6, 3, d, torch.bfloat16, device)
    lens = [keys, keys // 3]
    k[1, keys // 3:], v[1, keys // 3:] = NAN, INF
    assert plan(q, k)[2] > 1
    got = masked_attention(q, k, v, k_lengths=ints(lens, device), return_lse=True)
    check(got, definition(q, k, v, [(i, 0, rows, 0, n) for i, n in enumerate(lens)], scale=d ** -0.5))


@pytest.mark.parametrize("distance", [False, True])
@pytest.mark.parametrize("sq,sk,hq,hk", [(100, 200, 2, 2), (150, 333, 6, 2), (1, 3000, 14, 2), (1000, 1000, 74, 74)])
def test_masked_places_move_no_bit(device, sq, sk, hq, hk, distance):
    """Whatever keys and queries behind the sequences hold, under a cap: the same bits."""
    q, k, v = make(1, sq, sk, hq, hk, 128, torch.bfloat16, device)
    slopes = torch.exp2(-torch.arange(1, hq + 1, device=device).float() / hq) if distance else None
    nq, nk = max(sq * 2 // 3, 1), sk * 3 // 4 + 1
    for cap in (5.0, 40.0):
        want = None
        for fill in (0.0, 60.0, 3e38, NAN):
            q[:, nq:], k[:, nk:], v[:, nk:] = fill, fill, fill
            got = masked_attention(q, k, v, softcap=cap, slopes=slopes, q_lengths=ints([nq], device),
                                   k_lengths=ints([nk], device), return_lse=True)
            want = want or got
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("sq,sk,hq,hk", [(400, 400, 6, 2), (100, 64, 7, 1), (1000, 1000, 70, 10), (1, 3000, 24, 8)])
def test_unused_rows_of_a_tile_move_no_bit(device, sq, sk, hq, hk):
    """Rows that no query fills hold what an earlier kernel left in shared memory."""
    q, k, v = make(1, sq, sk, hq, hk, 128, torch.bfloat16, device)
    before = torch.zeros((1, 4096, 74, 128), device=device, dtype=torch.bfloat16)
    want = None
    for fill in (0.0, 30.0, NAN):
        before[:] = fill
        masked_attention(before, before[:, :64], before[:, :64])
        got = masked_attention(q, k, v, softcap=30.0, return_lse=True)
        want = want or got
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("distance", [False, True])
@pytest.mark.parametrize("lens,heads", [([40, 70, 18, 300, 128], 2), ([900, 30, 1200, 7, 900], 40)])
def test_other_documents_move_no_bit(device, lens, heads, distance):
    """Documents that share tiles and key blocks, under a cap: what one of them holds does not
    show in the others."""
    offs = [sum(lens[:i]) for i in range(len(lens) + 1)]
    q, k, v = make(1, offs[-1], offs[-1], heads, heads, 128, torch.bfloat16, device)
    slopes = torch.exp2(-torch.arange(1, heads + 1, device=device).float() / heads) if distance else None
    for cap in (5.0, 40.0):
        clean = masked_attention(q, k, v, q_offsets=ints(offs, device), k_offsets=ints(offs, device), softcap=cap,
                                 slopes=slopes, return_lse=True)
        for fill in (60.0, 3e38, NAN):
            a, b, c = q.clone(), k.clone(), v.clone()
            for t in (a, b, c):
                t[:, offs[1]:offs[2]], t[:, offs[3]:offs[4]] = fill, -fill
            got = masked_attention(a, b, c, q_offsets=ints(offs, device), k_offsets=ints(offs, device), softcap=cap,
                                   slopes=slopes, return_lse=True)
            for i in (0, 2, 4):
                rows = slice(offs[i], offs[i + 1])
                assert torch.equal(got[0][:, rows], clean[0][:, rows]) and torch.equal(got[1][..., rows], clean[1][..., rows])


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("sq,sk,n", [(2048, 2048, 2000), (1, 30000, 29950), (300, 16384, 16300)])
def test_padding_costs_nothing_by_what_it_holds(device, sq, sk, n, causal):
    """NaN behind the sequence takes no longer than zeros there (it took 14 times as long)."""
    q, k, v = make(1, sq, sk, 8, 8, 128, torch.bfloat16, device)
    lengths = ints([n], device)

    def ms():
        times = []
        for _ in range(7):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            for _ in range(5):
                masked_attention(q, k, v, k_lengths=lengths, causal=causal)
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end))
        return sorted(times)[3]
    v[:, n:] = 0
    clean, want = ms(), masked_attention(q, k, v, k_lengths=lengths, causal=causal)
    v[:, n:] = NAN
    assert ms() < 2 * clean
    assert torch.equal(masked_attention(q, k, v, k_lengths=lengths, causal=causal), want)


@pytest.mark.parametrize("form", ["rows", "pairs", "split"])
@pytest.mark.parametrize("d,t", [(128, torch.bfloat16), (64, torch.float16)])
def test_values_not_finite_at_both_ends(device, form, d, t):
    """V not finite at the first and the last key that rows see, NaN behind: it reaches the
    rows that see it, in its channel, and nothing else."""
    sq, sk, heads = dict(rows=(200, 700, 2), pairs=(1000, 1000, 74), split=(3, 20000, 2))[form]
    q, k, v = make(1, sq, sk, heads, heads, d, t, device)
    n = sk - 70
    lengths = ints([n], device)
    for causal in (False, True):
        v0 = v.clone()
        clean = masked_attention(q, k, v0, k_lengths=lengths, causal=causal)
        v0[0, 0, 0, 5], v0[0, n - 1, 1, 33], v0[0, n // 2, 0, 60], v0[0, n:] = INF, NAN, -INF, NAN
        out = masked_attention(q, k, v0, k_lengths=lengths, causal=causal)
        at = torch.arange(sq, device=device) + (n - sq if causal else sk)      # the last key a row sees
        want = clean.clone()
        want[0, at >= 0, 0, 5], want[0, at >= n - 1, 1, 33], want[0, at >= n // 2, 0, 60] = INF, NAN, -INF
        assert torch.equal(torch.isnan(out), torch.isnan(want))
        assert torch.equal(out.nan_to_num(5.0), want.nan_to_num(5.0))


def test_no_keys_of_any_layout(device):
    """An empty cache's strides and address are no one's business."""
    q = torch.randn((2, 5, 4, 128), device=device).bfloat16()
    buf = torch.empty((2, 9, 2, 133), device=device, dtype=torch.bfloat16)
    for none in (buf[:, :0, :, 1:129], buf[:, 9:, :, 3:131], torch.empty((2, 2, 0, 128), device=device, dtype=q.dtype).transpose(1, 2)):
        out, lse = masked_attention(q, none, none, return_lse=True)
        assert torch.all(out == 0) and torch.all(lse == -INF)


def test_patched_model_runs_the_provider(device):
    """A patched model's block gives the provider's result, by default too (verification against
    the block's own attention would put the original's in its place), and reports no fallback."""
    from h3_speedkit import synthetic
    from h3_speedkit.runtime import Backend, ModelPatch
    from test_gpu_attention import _h3_block_ns
    m, d, heads = 300, 512, 4
    bw = synthetic.cfg5_block(0, d, 1024, tables=2, device=device)
    block = _h3_block_ns(bw, *(torch.rand((2, 128), device=device) + 0.5).bfloat16())
    at = torch.arange(m, device=device, dtype=torch.int32)[:, None].repeat(1, 3)
    provider = MaskedAttentionProvider(heads, positions=at, sections=(16, 16, 16), causal=True)
    x, t_emb, segments = synthetic.cfg5_tokens(m, d, device=device), torch.zeros((1, 4), device=device), [(0, 100, 0), (100, m, 1)]
    backend = Backend()
    want = x.clone()
    backend.block(block, want, t_emb, segments, rows=(torch.arange(m, device=device) >= 100).int(), attention=provider)
    patch = ModelPatch(SimpleNamespace(blocks=[block]), backend, attention=provider, blocks=1)
    original = lambda inputs: {"img": torch.zeros_like(inputs["img"])}
    run = lambda x: patch.replacement(0)(dict(img=x, t_emb=t_emb, mod_segments=segments), dict(original_block=original))["img"]
    with torch.no_grad():
        for _ in range(2):
            got = patch.wrapper(run, x.clone())
            assert torch.equal(got, want)
            assert "fallback" not in patch.last_report and patch.last_report["counts"]["attention"] == 1


@pytest.mark.parametrize("sq,hq,hk,causal,documents,pairs", [
    (8192, 24, 24, False, 0, 0), (4096, 8, 8, False, 0, 0), (2048, 74, 74, False, 0, 0), (12288, 16, 4, False, 21, 0),
    (12288, 16, 4, False, 2, 0), (6000, 8, 2, True, 0, 0), (16384, 8, 8, False, 0, 0), (16384, 16, 16, False, 0, 1),
    (16384, 56, 56, False, 0, 1), (1000, 74, 74, False, 0, 1)])
def test_the_form_that_measured_shorter(device, sq, hq, hk, causal, documents, pairs):
    q = torch.empty((1, 1, 1, 128), device=device, dtype=torch.bfloat16)
    assert plan(q.expand(1, sq, hq, 128), q.expand(1, sq, hk, 128), documents, causal)[0] == pairs


@pytest.mark.parametrize("cap,distance", [(0.0, False), (30.0, True)])
@pytest.mark.parametrize("d,t", [(128, torch.bfloat16), (64, torch.float16)])
def test_many_single_tiles(device, cap, distance, d, t):
    """Long inputs whose tiles run singly, two to an SM, with every mask."""
    n, hq, hk = 1700, 28, 4
    q, k, v = make(1, n, n, hq, hk, d, t, device)
    slopes = torch.exp2(-0.1 * torch.arange(1, hq + 1, device=device)) if distance else None
    more, ref = dict(softcap=cap, slopes=slopes, return_lse=True), dict(scale=d ** -0.5, cap=cap, slopes=slopes)
    lens = [100, 0, 1, 600, 90, n - 791]
    offs = [sum(lens[:i]) for i in range(len(lens) + 1)]
    assert plan(q, k)[0] == 0 and plan(q, k, causal=True)[0] == 0 and plan(q, k, documents=len(lens))[0] == 0
    check(masked_attention(q, k, v, **more), definition(q, k, v, [(0, 0, n, 0, n)], **ref))
    check(masked_attention(q, k, v, causal=True, prefix=ints([333], device), **more),
          definition(q, k, v, [(0, 0, n, 0, n)], causal=True, prefix=[333], **ref))
    check(masked_attention(q, k, v, q_offsets=ints(offs, device), k_offsets=ints(offs, device), **more),
          definition(q, k, v, [(0, a, b, a, b) for a, b in zip(offs, offs[1:])], **ref))
