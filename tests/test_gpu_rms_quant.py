"""residual_rms_quant against the definition in 64 bits."""
import itertools

import pytest
import torch

from h3_speedkit.ops.gemm import int8_linear
from h3_speedkit.ops.rms_quant import residual_rms_quant

pytestmark = pytest.mark.gpu
EPS = 1e-6
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def definition(h, weight, dtype):
    """(y / scale before rounding, scale), both in 64 bits, from the stored h."""
    h, w = h.double(), weight.double()
    y = h / torch.sqrt(h.pow(2).mean(1, keepdim=True) + EPS) * w
    scale = (y.abs().amax(1, keepdim=True) / TOP[dtype]).clamp_min(1e-30)
    return y / scale, scale


def check(q, scale, h, weight, dtype):
    """Scales: a sum of K squares, its root and two products round within
    (log2-deep sums aside) K / threads + 40 half-steps at most, taken as 2e-6.  Codes:
    an exact y / s is off by at most that times 448, and the rounding by half a step."""
    exact, s = definition(h, weight, dtype)
    assert torch.all((scale.double() - s).abs() <= 2e-6 * s)
    codes = q.double()
    if dtype == torch.int8:
        assert torch.all((codes - exact).abs() <= 0.5 + 127 * 4e-6)
    else:
        # half a step of three bits behind the point: 2^-4 of the value, 2^-10 below 2^-6
        assert torch.all((codes - exact).abs() <= torch.maximum(exact.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10)) * 1.0001
                         + 448 * 4e-6)


def make(m, k, t, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed + m + k)
    x = torch.randn((m, k), generator=g, device=device).to(t)
    r = (torch.randn((m, k), generator=g, device=device) * 3).to(t)
    w = (1 + 0.2 * torch.randn(k, generator=g, device=device)).to(t)
    return x, r, w


@pytest.mark.parametrize("m,k", [(1, 1), (1, 7), (3, 8), (2, 31), (5, 256), (1, 264), (7, 1000), (130, 1155), (2, 4096),
                                 (9, 5376), (3, 8192), (2, 8200), (2, 16381), (3, 16384)])
@pytest.mark.parametrize("t,dtype,residual", list(itertools.product((torch.bfloat16, torch.float16),
                                                                   (torch.int8, torch.float8_e4m3fn), (False, True))))
def test_definition(device, m, k, t, dtype, residual):
    x, r, w = make(m, k, t, device)
    q, s, h = residual_rms_quant(x, w, residual=r if residual else None, dtype=dtype)
    assert q.dtype == dtype and tuple(s.shape) == (m, 1)
    if residual:
        assert torch.equal(h, (x.float() + r.float()).to(t))
    else:
        assert h is x
    check(q, s, h, w, dtype)


@pytest.mark.parametrize("offset,stride", [(0, 1040), (1, 1040), (8, 1031), (3, 1027)])
def test_strides_offsets_and_fp32_weight(device, offset, stride):
    m, k = 33, 1024
    x, r, w = make(m, stride + offset, torch.bfloat16, device)
    x, r = x[:, offset:offset + k], r[:, offset:offset + k]
    w = w[:k].float()
    q, s, h = residual_rms_quant(x, w, residual=r)
    assert torch.equal(h, (x.float() + r.float()).bfloat16())
    check(q, s, h, w, torch.int8)


@pytest.mark.parametrize("m,k", [(1, 9), (5, 63), (37, 1155), (3, 16384)])
@pytest.mark.parametrize("xo,ro,pad", [(0, 0, 1), (3, 3, 8), (1, 6, 16), (5, 0, 3)])
def test_operands_of_different_alignment(device, m, k, xo, ro, pad):
    x, r, w = make(m, k + pad + 8, torch.float16, device)
    keep_x, keep_r = x.clone(), r.clone()
    q, s, h = residual_rms_quant(x[:, xo:xo + k], w[:k], residual=r[:, ro:ro + k], dtype=torch.float8_e4m3fn)
    assert torch.equal(h, (x[:, xo:xo + k].float() + r[:, ro:ro + k].float()).half())
    check(q, s, h, w[:k], torch.float8_e4m3fn)
    assert torch.equal(x, keep_x) and torch.equal(r, keep_r)


@pytest.mark.parametrize("which", ["residual", "x"])
def test_in_place_stream(device, which):
    x, r, w = make(65, 640, torch.bfloat16, device)
    want = residual_rms_quant(x, w, residual=r)
    place = (r if which == "residual" else x).clone()
    args = (x, place) if which == "residual" else (place, r)
    got = residual_rms_quant(args[0], w, residual=args[1], residual_out=place)
    assert got[2] is place
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("which", ["residual", "x"])
def test_in_place_rows_of_odd_width(device, which):
    x, r, w = make(300, 643, torch.float16, device)
    want = residual_rms_quant(x, w, residual=r)
    assert torch.equal(want[2], (x.float() + r.float()).half())
    place = (r if which == "residual" else x).clone()
    args = (x, place) if which == "residual" else (place, r)
    got = residual_rms_quant(args[0], w, residual=args[1], residual_out=place)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_not_finite_rows_of_odd_width_stay_alone(device):
    x, _, w = make(9, 643, torch.float16, device)
    clean = residual_rms_quant(x, w)
    x = x.clone()
    x[2, -1], x[4, 0], x[7, 321] = float("nan"), float("inf"), float("-inf")
    q, s, _ = residual_rms_quant(x, w)
    bad = torch.tensor([2, 4, 7], device=device)
    assert torch.all(torch.isnan(s[bad]))
    keep = torch.tensor([0, 1, 3, 5, 6, 8], device=device)
    assert torch.equal(q[keep], clean[0][keep]) and torch.equal(s[keep], clean[1][keep])


def test_rows_without_values_zeros_and_not_finite(device):
    x, _, w = make(6, 512, torch.bfloat16, device)
    clean = residual_rms_quant(x, w)
    x = x.clone()
    x[1] = 0
    x[3, 17] = float("nan")
    x[4, 500] = float("inf")
    q, s, _ = residual_rms_quant(x, w)
    assert torch.all(q[1] == 0) and s[1].item() == pytest.approx(1e-30)
    assert torch.isnan(s[3]) and torch.isnan(s[4])
    for i in (0, 2, 5):
        assert torch.equal(q[i], clean[0][i]) and torch.equal(s[i], clean[1][i])
    q, s, h = residual_rms_quant(x[:0], w, residual=x[:0])
    assert q.shape == (0, 512) and s.shape == (0, 1) and h.shape == (0, 512)


def test_outputs_stream_and_graph(device):
    """The caller's outputs, a side stream, and a replayed graph on new values."""
    x, r, w = make(300, 4096, torch.bfloat16, device)
    want = residual_rms_quant(x, w, residual=r)
    out, scale, h = torch.empty_like(want[0]), torch.empty_like(want[1]), torch.empty_like(want[2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = residual_rms_quant(x, w, residual=r, out=out, out_scale=scale, residual_out=h)
    side.synchronize()
    assert got[0] is out and got[1] is scale and got[2] is h
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    xs = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = residual_rms_quant(xs, w, residual=r)
    xs.copy_(x.flip(0))
    graph.replay()
    again = residual_rms_quant(x.flip(0), w, residual=r)
    assert all(torch.equal(a, b) for a, b in zip(held, again))


def test_feeds_the_int8_linear(device):
    """norm -> codes -> INT8 product, against the product of the dequantised codes."""
    x, r, w = make(130, 512, torch.bfloat16, device)
    g = torch.Generator(device=device).manual_seed(1)
    wq = torch.randint(-127, 128, (256, 512), generator=g, device=device, dtype=torch.int8)
    ws = torch.rand(256, generator=g, device=device) * 1e-3 + 1e-4
    q, s, _ = residual_rms_quant(x, w, residual=r)
    out = int8_linear(q, wq, s, ws)
    want = (q.double() @ wq.double().T) * s.double() * ws.double()   # the integer sum is exact
    # one BF16 rounding of an FP32 value that was itself rounded three times
    assert torch.all((out.double() - want).abs() <= want.abs() * (2.0 ** -8 * 1.001))


def definition_at(h, weight, dtype, eps):
    h, w = h.double(), weight.double()
    y = h / torch.sqrt(h.pow(2).mean(1, keepdim=True) + eps) * w
    scale = (y.abs().amax(1, keepdim=True) / TOP[dtype]).clamp_min(1e-30)
    return y / scale, scale


FAR = [  # size of the values, of the FP32 weights, eps
    (1e25, 1.0, 1e-6), (3e38, 1.0, 1e-6), (1e25, 1.0, 3e38), (2e19, 1e-20, 1e-6), (1e18, 1e21, 1e-6), (1e30, 1e30, 1e-6),
    (1e-37, 1.0, 1e-20), (1e-37, 1.0, 1.2e-38), (3e-39, 1.0, 1.2e-38), (1e-10, 1e-30, 1e-30), (1e-25, 1e-15, 1.2e-38),
    (1e-37, 1e30, 1e-20), (1e-20, 1.0, 1e-6), (1e4, 1e-35, 1e-6)]


@pytest.mark.parametrize("size,by,eps", FAR)
@pytest.mark.parametrize("dtype", list(TOP))
@pytest.mark.parametrize("k", [1, 31, 256, 1155, 5376, 16381])
def test_values_far_from_one(device, size, by, eps, dtype, k):
    """Squares, products with the weights or the codes' factor that leave FP32's range, in
    every BF16 row that the formulas give finite values for; beside ordinary rows, whose
    bits do not change."""
    x, _, w = make(5, k, torch.bfloat16, device, seed=3)
    w, x = w.float() * by, x.float().clamp(-1, 1)
    x = x / x.abs().amax(1, keepdim=True)
    far = (x * size).to(torch.bfloat16)
    q, s, _ = residual_rms_quant(far, w, eps=eps, dtype=dtype)
    exact, want = definition_at(far, w, dtype, eps)
    assert torch.all((s.double() - want).abs() <= 2e-6 * want)
    # as in `check`: half a step of the codes, and the scale's part of a code
    half = 0.5 if dtype == torch.int8 else torch.maximum(exact.abs() * 2.0 ** -4 * 1.0001, torch.tensor(2.0 ** -10))
    assert torch.all((q.double() - exact).abs() <= half + TOP[dtype] * 4e-6)
    mixed = torch.cat((make(3, k, torch.bfloat16, device)[0], far))
    got = residual_rms_quant(mixed, w, eps=eps, dtype=dtype)
    alone = residual_rms_quant(mixed[:3].contiguous(), w, eps=eps, dtype=dtype)
    assert torch.equal(got[0][:3].view(torch.uint8), alone[0].view(torch.uint8)) and torch.equal(got[1][:3], alone[1])
    assert torch.equal(got[0][3:].view(torch.uint8), q.view(torch.uint8)) and torch.equal(got[1][3:], s)


@pytest.mark.parametrize("dtype", list(TOP))
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("eps", [1.2e-38, 1e-20, 1e-6, 3e38])
def test_zero_rows_at_any_epsilon(device, dtype, t, eps):
    for k in (64, 643):
        x = torch.zeros((4, k), device=device, dtype=t)
        x[2] = 1
        for w in (torch.ones(k, device=device), torch.ones(k, device=device, dtype=t), torch.zeros(k, device=device)):
            q, s, _ = residual_rms_quant(x, w, eps=eps, dtype=dtype)
            zero = slice(None) if not w.any() else torch.tensor([0, 1, 3], device=device)
            assert torch.all(q[zero].view(torch.uint8) == 0) and torch.all(s[zero] == torch.tensor(1e-30, device=device))


def test_large_rows_of_a_stream_in_place(device):
    """h beyond 2^64 in the caller's residual; and a row whose y passes FP32 is not finite."""
    for k in (640, 643):
        x, r, w = make(3, k, torch.bfloat16, device)
        x, r = (x.float() * 1e30).bfloat16(), (r.float() * 1e30).bfloat16()
        want = (x.float() + r.float()).bfloat16()
        q, s, h = residual_rms_quant(x, w, residual=r, residual_out=r)
        assert h is r and torch.equal(h, want)
        check(q, s, h, w, torch.int8)
        w = w.float()
        w[7] = 3e38
        x[1, 7] = 1e32
        assert torch.isnan(residual_rms_quant(x, w)[1][1])
