"""GPU: the 8-bit form and the activations that are kept in it (csrc/act_ckpt8.hip) against the definitions in 64 bits.

Tolerances: codes and scales are defined by exact arithmetic (a power of two, one rounding to nearest even), so they are compared for equality.
y and dh are rounded once (eps / 2 of themselves) after f32 arithmetic whose error is at most 24 * 2^-24 of max(1, |h|) times the factor in
front: the exponential's argument is off by 2^-24 of itself and the argument is below 16 * log2(e) wherever the result is above 2^-24, the
polynomial by 2^-21.  Column sums of n terms: 2^-24 * (sqrt(n) + 8) of the sum of magnitudes, plus the terms' own errors."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTS = {"relu": 1, "quickgelu": 2, "gelu": 3}
TOL = 24 * 2.0 ** -24


def _encode64(x, relu=False):
    """codes as values and scales, from the definition"""
    R, C = x.shape
    nb = (C + 31) // 32
    v = torch.zeros(R, nb * 32, dtype=torch.float64)
    v[:, :C] = x.double()
    v = v.view(R, nb, 32)
    a = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(-1)
    k = torch.full_like(a, -100.0)
    for e in range(-100, 121):                                    # the smallest power of two that will do
        k = torch.where(a > 448 * 2.0 ** (e - 1), torch.full_like(a, max(e, -100)), k)
    u = v / 2.0 ** k[..., None]
    step = 2.0 ** (torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))).clamp(min=-6) - 3)
    q = torch.where(torch.isfinite(u), torch.round(u / step) * step, torch.full_like(u, math.nan))
    if relu:
        q = torch.where(v <= 0, -q.abs(), q)
        q = torch.where(v == 0, torch.full_like(q, -0.0), q)
    return q.view(R, -1)[:, :C], 2.0 ** k


def _same_codes(ck, x, relu=False):
    q, s = _encode64(x, relu)
    c = ck.codes.cpu().double()
    assert torch.equal(ck.scales.cpu().double(), s)
    ok = (c == q) | (torch.isnan(c) & torch.isnan(q))
    assert ok.all(), (c[~ok][:5], q[~ok][:5])
    if relu:
        fine = torch.isfinite(q)
        assert torch.equal(torch.signbit(c)[fine], torch.signbit(q)[fine])


def _value8(ck):
    C = ck.codes.shape[1]
    return ck.codes.cpu().double() * ck.scales.cpu().double().repeat_interleave(32, 1)[:, :C]


def _act64(h, act):
    if act == "relu":
        return h.clamp(min=0), (~torch.signbit(h)).double()
    if act == "quickgelu":
        g = torch.sigmoid(1.702 * h)
        return h * g, g * (1 + 1.702 * h * (1 - g))
    phi = 0.5 * torch.special.erfc(-h / math.sqrt(2))
    return h * phi, phi + h * torch.exp(-h * h / 2) / math.sqrt(2 * math.pi)


def _inputs(rows, C, dt, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, C, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))).to(T[dt]), g


SHAPES = [(1, 1), (2, 3), (1, 31), (3, 32), (5, 33), (7, 96), (100, 257), (33, 511), (64, 512), (9, 513), (300, 1024), (4, 2048), (1500, 40),
          (2, 8200), (5001, 7)]


@pytest.mark.parametrize("rows,C", SHAPES)
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_encode_and_decode(rows, C, dt):
    from openvis_amd import ops
    x, _ = _inputs(rows, C, dt, rows + 31 * C)
    ck = ops.ckpt8_encode(x.cuda())
    assert ck.codes.shape == (rows, C) and ck.scales.shape == (rows, (C + 31) // 32)
    _same_codes(ck, x)
    for t in T.values():
        got = ops.ckpt8_decode(ck, t)
        assert got.dtype == t and torch.equal(got.cpu(), _value8(ck).float().to(t))


def test_every_code_rounding_and_limit():
    """all 16-bit patterns of bf16 and fp16 in blocks of their own scale, ties between codes, the largest and smallest blocks, NaN, infinities"""
    from openvis_amd import ops
    for t in (torch.bfloat16, torch.float16):
        x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(t).view(-1, 32)
        _same_codes(ops.ckpt8_encode(x.cuda()), x)
        one = x.view(-1, 1)                                       # a block each
        _same_codes(ops.ckpt8_encode(one.cuda()), one)
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (codes[1:] + codes[:-1]) / 2
    top = torch.full_like(mid, 448.0)                             # keeps the block's scale at 1
    for eps in (0.0, 2.0 ** -12, -2.0 ** -12):
        x = torch.stack((mid * (1 + eps), -mid * (1 + eps), top), 1).float()
        ck = ops.ckpt8_encode(x.cuda())
        assert (ck.scales.cpu().double() == 1).all()
        _same_codes(ck, x)
    x = torch.tensor([[448 * 2.0 ** k * f, 2.0 ** k, 0.0] for k in range(-120, 118) for f in (1.0, 1.0 + 2.0 ** -20, 1 - 2.0 ** -20)])
    x = torch.cat((x, torch.tensor([[0.0, -0.0, 0.0], [2.0 ** -149, 2.0 ** -126, 0.0], [3.4028234e38, 1.0, -3.4028234e38],
                                    [math.inf, 1.0, -2.0], [math.nan, 1.0, -2.0], [-math.inf, math.inf, math.nan], [math.nan, 0.0, 3e-3]])))
    _same_codes(ops.ckpt8_encode(x.cuda()), x)


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("rows,C", SHAPES)
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_forward_and_backward(rows, C, dt, act):
    from openvis_amd import ops
    h, g = _inputs(rows, C, dt, rows + 7 * C)
    dy = torch.randn(rows, C, generator=g).to(T[dt])
    y, ck = ops.act_forward_ckpt8(h.cuda(), ACTS[act])
    _same_codes(ck, h, act == "relu")
    half, tiny = torch.finfo(T[dt]).eps / 2, torch.finfo(T[dt]).tiny
    ry, _ = _act64(h.double(), act)
    assert y.dtype == T[dt]
    assert ((y.double().cpu() - ry).abs() <= half * ry.abs() * (1 + TOL) + TOL * h.double().abs().clamp(max=16) + tiny * half * 2).all()
    v = _value8(ck)
    ry, slope = _act64(v, act)
    for recompute in (False, True):
        dh, db, y8 = ops.act_backward_ckpt8(dy.cuda(), ck, ACTS[act], recompute=recompute)
        ref = dy.double() * slope
        err = half * ref.abs() * (1 + TOL) + TOL * 2 * dy.double().abs() + tiny * half * 2
        assert dh.dtype == T[dt] and ((dh.double().cpu() - ref).abs() <= err).all()
        bound = 2.0 ** -24 * (math.sqrt(rows) + 8) * ref.abs().sum(0) + TOL * 2 * dy.double().abs().sum(0) + 1e-30
        assert ((db.double().cpu() - ref.sum(0)).abs() <= bound).all()
        assert (y8 is not None) == recompute
        if recompute:
            w, scale = _value8(y8), y8.scales.cpu().double().repeat_interleave(32, 1)[:, :C]
            assert ((w - ry).abs() <= torch.maximum(ry.abs() * 2.0 ** -4, scale * 2.0 ** -10) * (1 + 1e-5) + TOL * v.abs().clamp(max=16)).all()


@pytest.mark.parametrize("act", list(ACTS))
def test_gradient_is_that_of_differences(act):
    """slope at the codes' values against central differences of the 64-bit activation"""
    from openvis_amd import ops
    h = torch.linspace(-6, 6, 1024).view(32, 32)
    _, ck = ops.act_forward_ckpt8(h.cuda(), ACTS[act])
    dh, _, _ = ops.act_backward_ckpt8(torch.ones(32, 32).cuda(), ck, ACTS[act])
    v, e = _value8(ck), 1e-5
    keep = v.abs() > 1e-3 if act == "relu" else torch.ones_like(v, dtype=torch.bool)
    diff = (_act64(v + e, act)[0] - _act64(v - e, act)[0]) / (2 * e)
    assert ((dh.double().cpu() - diff).abs()[keep] < 4e-6).all()


def test_relu_keeps_its_derivative_where_the_code_underflows():
    from openvis_amd import ops
    h = torch.tensor([[400.0, 1e-7, -1e-7, 0.0, -0.0, 2.0 ** -12, -3.0]]).cuda()
    _, ck = ops.act_forward_ckpt8(h, ops.ACT_RELU)
    dh, _, _ = ops.act_backward_ckpt8(torch.ones(1, 7).cuda(), ck, ops.ACT_RELU)
    assert dh.cpu().tolist() == [[1, 1, 0, 0, 0, 1, 0]]


def test_far_tails_and_not_finite_values():
    from openvis_amd import ops
    h = torch.tensor([[-60.0, -20.0, -9.0, 9.0, 20.0, 60.0, math.nan]] + [[x] * 7 for x in (1e4, -1e4)])
    for act in ("quickgelu", "gelu"):
        y, ck = ops.act_forward_ckpt8(h.cuda(), ACTS[act])
        ry = _act64(h.double(), act)[0]
        assert torch.isnan(y[0, 6]) and (y.cpu().double() - ry)[:, :6].abs().max() <= 2.0 ** -24 * 1e4
        dh, db, y8 = ops.act_backward_ckpt8(torch.ones(3, 7).cuda(), ck, ACTS[act], recompute=True)
        rs = _act64(_value8(ck), act)[1]
        assert (dh.cpu().double() - rs)[:, :6].abs().max() <= 2 * TOL and torch.isnan(dh[0, 6]) and torch.isnan(db[6]) and torch.isfinite(db[:6]).all()
        assert torch.isnan(y8.codes.float()[0, 6]) and torch.isfinite(y8.codes.float()[:, :6]).all()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_strided_rows(dt):
    from openvis_amd import ops
    x, g = _inputs(37, 411, dt, 5)
    h, dy = x.cuda()[:, 3:206], x.cuda()[:, 205:408]
    y, ck = ops.act_forward_ckpt8(h, ops.ACT_GELU)
    y2, ck2 = ops.act_forward_ckpt8(h.contiguous(), ops.ACT_GELU)
    assert torch.equal(y, y2) and torch.equal(ck.codes.view(torch.uint8), ck2.codes.view(torch.uint8))
    a, b = ops.act_backward_ckpt8(dy, ck, ops.ACT_GELU), ops.act_backward_ckpt8(dy.contiguous(), ck, ops.ACT_GELU)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_no_rows_streams_and_graphs():
    from openvis_amd import ops
    e = torch.empty(0, 48).cuda()
    y, ck = ops.act_forward_ckpt8(e, ops.ACT_GELU)
    dh, db, y8 = ops.act_backward_ckpt8(e, ck, ops.ACT_GELU, recompute=True)
    assert y.shape == dh.shape == (0, 48) and not db.any() and y8.codes.shape == (0, 48) and ops.ckpt8_decode(ck).shape == (0, 48)
    x, g = _inputs(3000, 1000, "f16", 2)
    x = x.cuda()

    def step():
        y, ck = ops.act_forward_ckpt8(x, ops.ACT_QUICKGELU)
        dh, db, y8 = ops.act_backward_ckpt8(x, ck, ops.ACT_QUICKGELU, recompute=True)
        return y, dh, db, y8.codes.view(torch.uint8)
    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        x.mul_(0.75)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step(), out)), k


def test_refusals():
    from openvis_amd import ops
    from openvis_amd._lib import OvisError
    x = torch.zeros(4, 64).cuda()
    _, ck = ops.act_forward_ckpt8(x, 3)
    bad = [lambda: ops.act_forward_ckpt8(x, 0), lambda: ops.act_forward_ckpt8(x, 4), lambda: ops.act_forward_ckpt8(x.double(), 3),
           lambda: ops.act_forward_ckpt8(x.cpu(), 3), lambda: ops.act_forward_ckpt8(x.t(), 3), lambda: ops.ckpt8_encode(x.int()),
           lambda: ops.act_backward_ckpt8(x, ck, 0), lambda: ops.act_backward_ckpt8(x[:3], ck, 3), lambda: ops.act_backward_ckpt8(x[:, :32], ck, 3),
           lambda: ops.act_backward_ckpt8(x.double(), ck, 3), lambda: ops.ckpt8_decode(ck, torch.float64),
           lambda: ops.ckpt8_decode(ops.Ckpt8(ck.codes, ck.scales[:3])), lambda: ops.ckpt8_decode(ops.Ckpt8(ck.codes.view(torch.uint8), ck.scales)),
           lambda: ops.ckpt8_decode(ops.Ckpt8(ck.codes.cpu(), ck.scales))]
    for f in bad:
        with pytest.raises(OvisError):
            f()
