"""rope_axes and rope_table against complex rotations in 64 bits."""
import pytest
import torch

from h3_speedkit.ops.rope import rope_axes, rope_table

pytestmark = pytest.mark.gpu
EPS = 1e-6


def angles(positions, sections, theta):
    thetas = theta if isinstance(theta, tuple) else (theta,) * len(sections)
    cols = [positions[:, a].double() * thetas[a] ** (-i / n) for a, n in enumerate(sections) for i in range(n)]
    return torch.stack(cols, 1)


def definition(x, positions, sections, theta, interleaved, weight=None, sign=1.0):
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * weight.double()
    a = angles(positions, sections, theta) * sign
    z, n, y = torch.polar(torch.ones_like(a), a)[:, None], a.shape[1], x.clone()
    if interleaved:
        r = torch.complex(x[..., 0:2 * n:2].contiguous(), x[..., 1:2 * n:2].contiguous()) * z
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = r.real, r.imag
    else:
        r = torch.complex(x[..., :n].contiguous(), x[..., n:2 * n].contiguous()) * z
        y[..., :n], y[..., n:2 * n] = r.real, r.imag
    return y


def close(got, want, scale):
    """Half a step of the type, and FP32's part: six roundings of terms below the row's
    largest value (the pair's length at most sqrt 2 of it)."""
    half = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0    # half a step of FP16's subnormals
    err = (got.double() - want).abs()
    assert torch.all(err <= half * want.abs() * 1.001 + scale * 2e-6 + tiny), float(err.max())


def make(tokens, hq, hk, dim, t, device, axes=3, whole=True, seed=0):
    g = torch.Generator(device=device).manual_seed(seed + tokens)
    qkv = torch.randn((tokens, (hq + 2 * hk) * dim), generator=g, device=device).to(t)
    q, k = qkv[:, :hq * dim].view(tokens, hq, dim), qkv[:, hq * dim:(hq + hk) * dim].view(tokens, hk, dim)
    at = torch.rand((tokens, axes), generator=g, device=device) * torch.tensor([5000.0, 90.0, 160.0][:axes], device=device)
    return q, k, at.floor().int() if whole else at, qkv


@pytest.mark.parametrize("tokens,hq,hk", [(1, 56, 56), (1, 1, 1), (5, 3, 1), (129, 24, 8), (1000, 2, 2), (17, 130, 5)])
@pytest.mark.parametrize("dim,sections", [(128, (16, 16, 16)), (128, (24, 20, 20)), (64, (7, 9, 11)), (64, (32,)), (96, (24, 24)),
                                          (256, (128,)), (2, (1,)), (80, (8, 0, 24)), (160, (40, 8)), (34, (3, 3))])
@pytest.mark.parametrize("interleaved", [False, True])
def test_definition(device, tokens, hq, hk, dim, sections, interleaved):
    for t, whole, norm in ((torch.bfloat16, True, True), (torch.float16, False, False), (torch.bfloat16, False, False)):
        q, k, at, _ = make(tokens, hq, hk, dim, t, device, len(sections), whole)
        qw, kw = (1 + 0.2 * torch.randn(2, dim, device=device)).to(t) if norm else (None, None)
        qo, ko = rope_axes(q, k, at, sections=sections, interleaved=interleaved, q_weight=qw, k_weight=kw)
        for x, w, got in ((q, qw, qo), (k, kw, ko)):
            want = definition(x, at, sections, 10000.0, interleaved, w)
            close(got, want, want.abs().amax(-1, keepdim=True) * 2)


def test_far_positions_thetas_and_fp32_weights(device):
    """Angles keep their fraction at positions of 2^31; every axis has its own theta."""
    q, k, _, _ = make(8, 4, 2, 128, torch.float16, device)
    top = 2 ** 31 - 1
    at = torch.tensor([[top, -top - 1, 0], [top - 1, 7, 3], [1, 2, 3], [0, 0, 0], [10 ** 9, -5, 2 ** 30], [-1, -2, -3],
                       [65536, 65537, 99999], [123456789, 987654321, 5]], dtype=torch.int32, device=device)
    w = 1 + 0.1 * torch.rand(128, device=device)
    theta = (500.0, 10000.0, 1e6)
    qo, ko = rope_axes(q, k, at, sections=(24, 20, 20), theta=theta, q_weight=w, k_weight=w)
    for x, got in ((q, qo), (k, ko)):
        want = definition(x, at, (24, 20, 20), theta, False, w)
        close(got, want, want.abs().amax(-1, keepdim=True) * 2)


def test_inverse_is_the_gradient(device):
    """The inverse turns back, and equals the gradient of <rope(x), u> by differences."""
    q, k, at, _ = make(40, 4, 2, 64, torch.float16, device)
    u = torch.randn_like(q)
    back, _ = rope_axes(u, None, at, sections=(8, 8, 8), inverse=True)
    close(back, definition(u, at, (8, 8, 8), 10000.0, False, sign=-1.0), u.abs().amax(-1, keepdim=True).double() * 2)
    # the map is linear: f(q + e d) - f(q) over e is <rope(d), u>, whatever e is
    d = torch.randn(q.shape, device=device, dtype=torch.float64)
    step = (definition(q.double() + 0.5 * d, at, (8, 8, 8), 10000.0, False) -
            definition(q.double(), at, (8, 8, 8), 10000.0, False)) / 0.5
    left, right = (step * u.double()).sum(), (d * back.double()).sum()
    # half a step of each gradient value, added up at the worst
    assert abs(left - right) <= (d.abs() * back.double().abs()).sum() * 2.0 ** -11 + 1e-3


def test_in_place_slices_of_a_projection(device):
    """Q and K rotated where they lie in one projection: V and the gaps stay."""
    q, k, at, qkv = make(77, 6, 2, 128, torch.bfloat16, device)
    kept, (qw, kw) = qkv.clone(), (1 + 0.2 * torch.randn(2, 128, device=device)).bfloat16()
    want = rope_axes(q, k, at, sections=(16, 16, 16), q_weight=qw, k_weight=kw)
    got = rope_axes(q, k, at, sections=(16, 16, 16), q_weight=qw, k_weight=kw, q_out=q, k_out=k)
    assert got[0] is q and got[1] is k
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(qkv[:, 8 * 128:], kept[:, 8 * 128:])


def test_misaligned_and_strided(device):
    buf = torch.randn((50, 9, 131), device=device).bfloat16()
    q = buf[:, 1:8, 3:131]
    at = torch.arange(50, device=device, dtype=torch.int32)[:, None].contiguous()
    w = torch.rand(129, device=device).bfloat16()[1:]
    qo, none = rope_axes(q, None, at, sections=(48,), q_weight=w)
    assert none is None
    want = definition(q, at, (48,), 10000.0, False, w)
    close(qo, want, want.abs().amax(-1, keepdim=True) * 2)
    one = q[:, :1].expand(50, 7, 128)          # shared heads
    assert torch.equal(rope_axes(one, None, at, sections=(48,))[0], rope_axes(one.contiguous(), None, at, sections=(48,))[0])


@pytest.mark.parametrize("tokens", [0, 1, 333, 100000])
@pytest.mark.parametrize("sections", [(16, 16, 16), (5,), (64, 64)])
def test_table(device, tokens, sections):
    _, _, at, _ = make(tokens, 1, 1, 2, torch.bfloat16, device, len(sections))
    table = rope_table(at, sections=sections)
    assert tuple(table.shape) == (1, tokens, 1, sum(sections), 2, 2)
    a = angles(at, sections, 10000.0)
    want = torch.stack((a.cos(), -a.sin(), a.sin(), a.cos()), -1).view(table.shape)
    err = (table.double() - want).abs()
    # half a step; an angle off by 2^-22 turns moves a sine by 1.5e-6
    assert torch.all(err <= want.abs() * (2.0 ** -8 * 1.001) + 2e-6)


def test_table_drives_the_qkv_op(device):
    """The table has the QKV op's layout: its roped Q plane equals rope_axes with the norm
    (BF16 roundings in between differ, so within two steps and a rounding of the table)."""
    from h3_speedkit.ops.qkv import QKV
    m, heads, hidden = 40, 2, 256
    g = torch.Generator(device=device).manual_seed(3)
    q = torch.randint(-127, 128, (m, hidden), generator=g, device=device, dtype=torch.int8)
    w = torch.randint(-127, 128, (3 * heads * 128, hidden), generator=g, device=device, dtype=torch.int8)
    xs, ws = torch.rand((m, 1), generator=g, device=device) * 1e-2 + 1e-3, torch.full((3 * heads * 128, 1), 1e-2, device=device)
    weight = (1 + 0.1 * torch.rand(128, generator=g, device=device)).bfloat16()
    at = torch.randint(0, 500, (m, 3), generator=g, device=device, dtype=torch.int32)
    out = QKV().run(q, w, xs, ws, rope_table(at, sections=(16, 16, 16)), weight, weight, 1e-6)
    plain = ((q.double() @ w.double().T) * xs.double() * ws.double().T).bfloat16()[:, :heads * 128].view(m, heads, 128)
    want, _ = rope_axes(plain, None, at, sections=(16, 16, 16), q_weight=weight)
    got = out["d"][0].transpose(0, 1).double()
    # the op rounds x * rrms, its product with the weight, and the result to BF16, and reads
    # BF16 sines: each off by 2^-8 at most of a value no larger than the head's largest
    assert torch.all((got - want.double()).abs() <= want.double().abs().amax(-1, keepdim=True) * 6 * 2.0 ** -8)


def test_stream_and_graph(device):
    q, k, at, _ = make(500, 8, 8, 128, torch.bfloat16, device)
    want = rope_axes(q, k, at, sections=(16, 16, 16))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rope_axes(q, k, at, sections=(16, 16, 16))
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    held_at, graph = at.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = rope_axes(q, k, held_at, sections=(16, 16, 16))
        table = rope_table(held_at, sections=(16, 16, 16))
    held_at.copy_(at.flip(0))
    graph.replay()
    again = rope_axes(q, k, at.flip(0).contiguous(), sections=(16, 16, 16))
    assert all(torch.equal(a, b) for a, b in zip(held, again))
    assert torch.equal(table, rope_table(held_at, sections=(16, 16, 16)))


@pytest.mark.parametrize("size", [1e-30, 1e18, 1e19, 1e25, 3e38])
@pytest.mark.parametrize("dim,sections,interleaved", [(128, (16, 16, 16), False), (64, (7, 9, 11), True), (256, (128,), False),
                                                      (34, (3, 3), False), (128, (5,), False)])
def test_norm_of_heads_of_any_size(device, size, dim, sections, interleaved):
    """Squares past FP32 beside ordinary heads, whose bits do not change."""
    q, k, at, _ = make(37, 5, 2, dim, torch.bfloat16, device, len(sections))
    qw, kw = (1 + 0.2 * torch.randn(2, dim, device=device)).bfloat16()
    go = lambda q: rope_axes(q, k, at, sections=sections, interleaved=interleaved, q_weight=qw, k_weight=kw)
    plain = go(q)
    far = q.float() / q.float().abs().amax(-1, keepdim=True) * size
    mixed = q.clone()
    mixed[:, ::2] = far[:, ::2].bfloat16()
    got = go(mixed)
    want = definition(mixed, at, sections, 10000.0, interleaved, qw)
    close(got[0], want, want.abs().amax(-1, keepdim=True) * 2)
    assert torch.equal(got[0][:, 1::2], plain[0][:, 1::2]) and torch.equal(got[1], plain[1])
    mixed[3, 1, 2], mixed[4, 0, 1] = float("nan"), float("inf")
    bad = go(mixed)[0]
    assert torch.isnan(bad[3, 1]).all() and torch.isnan(bad[4, 0]).any()
    bad[3, 1], bad[4, 0] = got[0][3, 1], got[0][4, 0]
    assert torch.equal(bad, got[0])


@pytest.mark.parametrize("tokens,hq,hk", [(70, 6, 2), (1500, 6, 2), (2500, 6, 2), (300, 60, 52), (700, 130, 70), (9000, 60, 52),
                                          (17000, 60, 52), (16500, 20, 12)])
@pytest.mark.parametrize("dim,sections,norm", [(128, (16, 16, 16), True), (64, (7, 9, 11), False)])
def test_a_call_is_its_tokens_calls(device, tokens, hq, hk, dim, sections, norm):
    """However the rows are cut into tiles: the bits of calls on pieces of the tokens and heads."""
    q, k, at, _ = make(tokens, hq, hk, dim, torch.bfloat16, device, len(sections))
    w = (1 + 0.2 * torch.randn(dim, device=device)).bfloat16() if norm else None
    whole = rope_axes(q, k, at, sections=sections, q_weight=w, k_weight=w)
    for cut in (slice(0, 1), slice(tokens // 3, tokens // 3 + 65), slice(tokens - 40, None)):
        part = rope_axes(q[cut], None, at[cut].contiguous(), sections=sections, q_weight=w)[0]
        assert torch.equal(part, whole[0][cut])
        part = rope_axes(q[cut, :1], k[cut, -1:], at[cut].contiguous(), sections=sections, q_weight=w, k_weight=w)
        assert torch.equal(part[0], whole[0][cut, :1]) and torch.equal(part[1], whole[1][cut, -1:])
