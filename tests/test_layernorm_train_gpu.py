"""GPU: layer norm for training (csrc/layernorm_train.hip) against the formulas in 64 bits.

Tolerances: an output rounded once to a type of step eps is off by eps / 2 of itself.  The f32 arithmetic in front of it adds, relative to the
row's largest value, a few roundings (2^-24 each) of xhat, gamma and the sums of C terms, whose errors grow with the square root of C at
random; 64 * 2^-24 covers C = 8192.  dgamma / dbeta are sums of n = rows terms in f32: 2^-24 * (sqrt(n) + 8) of the sum of the magnitudes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32 = 64 * 2.0 ** -24
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _half(dt):
    return torch.finfo(dt).eps / 2


def _make(rows, C, xt, yt, seed, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, C, generator=g) * (1 + 3 * torch.rand(C, generator=g)) + offset).to(T[xt])
    gamma = 1 + 0.3 * torch.randn(C, generator=g)
    beta = 0.3 * torch.randn(C, generator=g)
    dy = torch.randn(rows, C, generator=g).to(T[yt])
    return x, gamma, beta, dy, g


def _forward64(s, gamma, beta, eps=1e-5):
    s = s.double()
    mean = s.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((s - mean).pow(2).mean(1, keepdim=True) + eps)
    xhat = (s - mean) * rstd
    return xhat * gamma.double() + beta.double(), xhat, mean, rstd


def _backward64(dy, xhat, rstd, gamma, dsum=None):
    dy, gd = dy.double(), dy.double() * gamma.double()
    dx = rstd * (gd - gd.mean(1, keepdim=True) - xhat * (gd * xhat).mean(1, keepdim=True))
    return dx if dsum is None else dx + dsum.double(), (dy * xhat).sum(0), dy.sum(0)


def _close(out, ref, dt, what, f32=F32):
    out, ref = out.double().cpu(), ref.cpu()
    scale = ref.abs().amax(-1, keepdim=True) + 1e-30
    bad = (out - ref).abs() > _half(dt) * ref.abs() * (1 + f32) + f32 * scale + torch.finfo(dt).tiny * _half(dt) * 2
    assert not bad.any(), (what, (out - ref).abs().max().item(), int(bad.sum()))


def _sum_close(out, ref, mag, n, what):
    assert ((out.double().cpu() - ref).abs() <= 2.0 ** -24 * (math.sqrt(n) + 8) * mag + 1e-30).all(), what


def _value8(ck):
    C = ck.codes.shape[1]
    return ck.codes.cpu().double() * ck.scales.cpu().double().repeat_interleave(32, 1)[:, :C]


SHAPES = [(1, 1), (3, 2), (1, 7), (5, 31), (9, 33), (100, 256), (64, 128), (33, 191), (7, 192), (17, 384), (130, 512), (300, 768), (3, 1000),
          (2051, 257), (5, 1536), (31, 2047), (6, 2049), (12, 4096), (3, 5001), (2, 8192), (701, 2600), (300, 2051), (1501, 1111), (37, 3500), (900, 6150)]


@pytest.mark.parametrize("rows,C", SHAPES)
@pytest.mark.parametrize("xt,yt", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")])
def test_forward_and_backward(rows, C, xt, yt):
    from openvis_amd import ops
    x, gamma, beta, dy, g = _make(rows, C, xt, yt, rows * 8191 + C)
    res = torch.randn(rows, C, generator=g).to(T[xt])
    dsum = torch.randn(rows, C, generator=g).to(T[xt])
    for r, ds in ((None, None), (res, dsum)):
        o = ops.layernorm_forward(x.cuda(), gamma.cuda(), beta.cuda(), residual=None if r is None else r.cuda(), out_dtype=T[yt])
        s = x if r is None else (x.float() + r.float()).to(T[xt])
        assert torch.equal(o.sum.cpu(), s) and o.y.dtype == T[yt] and o.xhat8 is None
        y, xhat, mean, rstd = _forward64(s, gamma, beta)
        # xhat of a row whose spread is small against its mean loses |mean| / spread of f32's precision
        lift = 1 + (mean.abs() * rstd).max().item()
        _close(o.y, y, T[yt], "y", F32 * lift)
        assert torch.allclose(o.stats[:, :1].double().cpu(), mean, rtol=0, atol=8 * 2.0 ** -24 * s.double().abs().max().item())
        assert torch.allclose(o.stats[:, 1:].double().cpu(), rstd, rtol=F32 * lift)
        # backward from these statistics, as a user has them
        st = o.stats.double().cpu()
        xh = (s.double() - st[:, :1]) * st[:, 1:]
        dx, dg, db = ops.layernorm_backward(dy.cuda(), o.sum, o.stats, gamma.cuda(), dsum=None if ds is None else ds.cuda())
        rx, rg, rb = _backward64(dy, xh, st[:, 1:], gamma, ds)
        part = _backward64(dy, xh, st[:, 1:], gamma)[0].abs().amax(1, keepdim=True) + (st[:, 1:] * (dy.double() * gamma.double()).abs().amax(1, keepdim=True))
        bad = (dx.double().cpu() - rx).abs() > _half(T[xt]) * rx.abs() * (1 + F32) + F32 * lift * (1 + xh.abs().max()) * part + torch.finfo(T[xt]).tiny * _half(T[xt]) * 2
        assert dx.dtype == T[xt] and not bad.any(), (dx.double().cpu() - rx).abs().max()
        _sum_close(dg, rg, (dy.double() * xh).abs().sum(0) * lift, rows, "dgamma")
        _sum_close(db, rb, dy.double().abs().sum(0), rows, "dbeta")


@pytest.mark.parametrize("rows,C", [(1, 1), (3, 31), (5, 33), (100, 256), (50, 257), (40, 768), (3, 2500), (2, 8191), (701, 2600), (300, 2051), (301, 1100), (40, 3501)])
@pytest.mark.parametrize("xt,yt", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16")])
def test_checkpoint_in_8_bits(rows, C, xt, yt):
    from openvis_amd import ops
    x, gamma, beta, dy, g = _make(rows, C, xt, yt, rows + 100 * C)
    dsum = torch.randn(rows, C, generator=g).to(T[xt])
    o = ops.layernorm_forward(x.cuda(), gamma.cuda(), beta.cuda(), out_dtype=T[yt], checkpoint=True)
    plain = ops.layernorm_forward(x.cuda(), gamma.cuda(), beta.cuda(), out_dtype=T[yt])
    assert torch.equal(o.y, plain.y) and torch.equal(o.stats, plain.stats)
    _, xhat, mean, rstd = _forward64(x, gamma, beta)
    v, scale = _value8(o.xhat8), o.xhat8.scales.cpu().double().repeat_interleave(32, 1)[:, :C]
    lift = 1 + (mean.abs() * rstd).max().item()
    # half a step: 2^-4 of the value, or 2^-10 of the scale below 2^-6 of it; and the f32 error of xhat itself
    assert ((v - xhat).abs() <= torch.maximum(xhat.abs() * 2.0 ** -4, scale * 2.0 ** -10) + 2 * F32 * lift * (1 + xhat.abs().max())).all()
    dx, dg, db = ops.layernorm_backward(dy.cuda(), o.xhat8, o.stats, gamma.cuda(), dsum=dsum.cuda())
    st = o.stats.double().cpu()
    rx, rg, rb = _backward64(dy, v, st[:, 1:], gamma, dsum)
    part = (st[:, 1:] * (dy.double() * gamma.double()).abs().amax(1, keepdim=True)) * (1 + v.abs().max()) ** 2
    assert dx.dtype == T[xt]
    assert ((dx.double().cpu() - rx).abs() <= _half(T[xt]) * rx.abs() * (1 + F32) + F32 * part + torch.finfo(T[xt]).tiny * _half(T[xt]) * 2).all()
    _sum_close(dg, rg, (dy.double() * v).abs().sum(0), rows, "dgamma")
    _sum_close(db, rb, dy.double().abs().sum(0), rows, "dbeta")


def test_gradients_are_those_of_differences():
    """dx, dgamma, dbeta against central differences of the 64-bit forward: (f(p + h) - f(p - h)) / 2h is off by h^2 f''' / 6 and 2^-52 |f| / h"""
    from openvis_amd import ops
    rows, C, h = 3, 40, 1e-4
    x, gamma, beta, dy, g = _make(rows, C, "f32", "f32", 3)
    o = ops.layernorm_forward(x.cuda(), gamma.cuda(), beta.cuda())
    dx, dg, db = [t.double().cpu() for t in ops.layernorm_backward(dy.cuda(), x.cuda(), o.stats, gamma.cuda())]
    f = lambda x_, g_, b_: (_forward64(x_, g_, b_)[0] * dy.double()).sum()
    for k in range(0, rows * C, 7):
        e = torch.zeros(rows * C, dtype=torch.float64)
        e[k] = h
        e = e.view(rows, C)
        assert abs(((f(x.double() + e, gamma, beta) - f(x.double() - e, gamma, beta)) / (2 * h)).item() - dx.view(-1)[k].item()) < 1e-5
    for k in range(0, C, 5):
        e = torch.zeros(C, dtype=torch.float64)
        e[k] = h
        assert abs(((f(x, gamma.double() + e, beta) - f(x, gamma.double() - e, beta)) / (2 * h)).item() - dg[k].item()) < 1e-5
        assert abs(((f(x, gamma, beta.double() + e) - f(x, gamma, beta.double() - e)) / (2 * h)).item() - db[k].item()) < 1e-5


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_strided_rows_and_offsets(dt):
    """rows that are a slice of wider ones, starting at any element: the same bits as the dense rows"""
    from openvis_amd import ops
    rows, C = 37, 203
    x, gamma, beta, dy, g = _make(rows, 3 * C + 5, dt, dt, 9)
    gamma, beta = gamma[:C].contiguous().cuda(), beta[:C].contiguous().cuda()
    xs, rs = x.cuda()[:, 1:1 + C], dy.cuda()[:, C + 2:2 * C + 2]
    a = ops.layernorm_forward(xs, gamma, beta, residual=rs, checkpoint=True)
    b = ops.layernorm_forward(xs.contiguous(), gamma, beta, residual=rs.contiguous(), checkpoint=True)
    for p, q in ((a.y, b.y), (a.sum, b.sum), (a.stats, b.stats), (a.xhat8.codes.view(torch.uint8), b.xhat8.codes.view(torch.uint8))):
        assert torch.equal(p, q)
    p = ops.layernorm_backward(rs, xs, a.stats, gamma, dsum=xs)
    q = ops.layernorm_backward(rs.contiguous(), xs.contiguous(), a.stats, gamma, dsum=xs.contiguous())
    assert all(torch.equal(u, v) for u, v in zip(p, q))
    cls = x.cuda().view(1, rows, -1)[:, 4, :C]                    # a class-token row: [1, C] with a wide stride
    assert torch.equal(ops.layernorm_forward(cls, gamma, beta).y, ops.layernorm_forward(cls.contiguous(), gamma, beta).y)


def test_large_offsets_constant_rows_and_not_finite_rows():
    from openvis_amd import ops
    C = 96
    gamma, beta = torch.full((C,), 2.0).cuda(), torch.full((C,), 0.5).cuda()
    x = torch.zeros(6, C)
    x[1] = 1e4 + torch.linspace(-1, 1, C)                         # mean far from 0: two passes keep the spread
    x[2, 3], x[3, 5] = math.inf, math.nan
    x[4] = torch.linspace(-1, 1, C)
    x[5] = torch.linspace(-1, 1, C) * 1e18
    o = ops.layernorm_forward(x.cuda(), gamma, beta, checkpoint=True)
    y = o.y.cpu()
    assert torch.equal(y[0], torch.full((C,), 0.5))               # a constant row: xhat = 0
    assert (y[1].double() - (_forward64(x[1:2], gamma.cpu(), beta.cpu())[0])[0]).abs().max() < 1e4 * 2.0 ** -22
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all()
    assert torch.isfinite(y[[0, 1, 4, 5]]).all()
    assert torch.isnan(o.xhat8.codes.float().cpu()[2]).all() and torch.isfinite(o.xhat8.codes.float().cpu()[[0, 1, 4, 5]]).all()
    dy = torch.ones(6, C).cuda()
    dx, dg, db = ops.layernorm_backward(dy, x.cuda(), o.stats, gamma)
    assert torch.isfinite(dx.cpu()[[0, 1, 4, 5]]).all() and torch.isnan(dx.cpu()[2]).any()
    assert torch.equal(db.cpu(), torch.full((C,), 6.0))


def test_no_rows():
    from openvis_amd import ops
    g = torch.ones(64).cuda()
    x = torch.empty(0, 64).cuda()
    o = ops.layernorm_forward(x, g, g, checkpoint=True)
    assert o.y.shape == (0, 64) and o.stats.shape == (0, 2) and o.xhat8.scales.shape == (0, 2)
    dx, dg, db = ops.layernorm_backward(x, x, o.stats, g)
    assert dx.shape == (0, 64) and not dg.any() and not db.any()


def test_same_bits_on_another_stream_and_in_a_replayed_graph():
    from openvis_amd import ops
    x, gamma, beta, dy, g = [t.cuda() if torch.is_tensor(t) else t for t in _make(5000, 768, "f16", "f16", 1)]

    def step():
        o = ops.layernorm_forward(x, gamma, beta, checkpoint=True)
        return (o.y, o.stats) + ops.layernorm_backward(dy, o.xhat8, o.stats, gamma, dsum=dy)
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
        x.mul_(1.25)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step(), out)), k


def test_refusals():
    from openvis_amd import ops
    from openvis_amd._lib import OvisError
    x, g = torch.zeros(4, 64).cuda(), torch.ones(64).cuda()
    st = torch.zeros(4, 2).cuda()
    bad = [lambda: ops.layernorm_forward(x.double(), g, g), lambda: ops.layernorm_forward(x.cpu(), g, g), lambda: ops.layernorm_forward(x, g[:32], g),
           lambda: ops.layernorm_forward(x, g.half(), g), lambda: ops.layernorm_forward(x, g, g, residual=x.half()),
           lambda: ops.layernorm_forward(x.half(), g, g, out_dtype=torch.float32), lambda: ops.layernorm_forward(x.t(), g[:4].contiguous(), g[:4].contiguous()),
           lambda: ops.layernorm_forward(x[:1].expand(4, 64), g, g), lambda: ops.layernorm_forward(torch.zeros(2, 8193).cuda(), torch.ones(8193).cuda(), torch.ones(8193).cuda()),
           lambda: ops.layernorm_backward(x, x[:3], st, g), lambda: ops.layernorm_backward(x, x, st[:3], g), lambda: ops.layernorm_backward(x, x.half(), st, g),
           lambda: ops.layernorm_backward(x, x, st, g, dsum=x.half()), lambda: ops.layernorm_backward(x, ops.Ckpt8(x, x), st, g),
           lambda: ops.layernorm_backward(x, x, st, g, out_dtype=torch.float16)]
    for f in bad:
        with pytest.raises(OvisError):
            f()
