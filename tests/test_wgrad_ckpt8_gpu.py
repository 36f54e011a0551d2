"""GPU: a linear layer's weight and bias gradient from its 8-bit input (csrc/wgrad_ckpt8.hip) against 64 bits.

Tolerances: products are exact (bf16, fp16: 4 significant bits of x by 8 or 11 of dy; f32: dy as a sum of three bf16 numbers, 2^-24 of it), sums
are f32.  A matrix instruction adds 16 products at a time to its accumulator: n = M / 16 roundings, each 2^-23 of the partial sum at most
(truncation), which random terms bring to 2^-23 * (sqrt(M / 16) + 16) of the sum of the magnitudes; all-of-one-sign sums to 2^-23 * M / 16."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _value8(ck):
    C = ck.codes.shape[1]
    return ck.codes.cpu().double() * ck.scales.cpu().double().repeat_interleave(32, 1)[:, :C]


SHAPES = [(1, 1, 1), (1, 3, 5), (7, 8, 32), (63, 64, 64), (64, 65, 33), (65, 33, 65), (100, 256, 2048), (197, 129, 257), (300, 100, 1000), (1000, 64, 48),
          (4097, 72, 200), (5000, 384, 96), (20000, 8, 16), (2500, 768, 768), (9000, 1030, 520), (33000, 256, 512), (9000, 2048, 2100), (70001, 1000, 1000)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_against_64_bits(M, N, K, dt):
    from openvis_amd import ops
    g = torch.Generator().manual_seed(M + N + K)
    x = torch.randn(M, K, generator=g) * torch.exp(torch.randn(K, generator=g)) * torch.exp(torch.randn(M, 1, generator=g))
    dy = (torch.randn(M, N, generator=g) * torch.exp(torch.randn(N, generator=g))).to(T[dt])
    gamma, beta = torch.randn(K, generator=g), torch.randn(K, generator=g)
    x8 = ops.ckpt8_encode(x.cuda())
    v, d = _value8(x8).cuda(), dy.double().cuda()
    ref, mag, rb, mb = d.t() @ v, d.abs().t() @ v.abs(), d.sum(0), d.abs().sum(0)
    tol, tolb = 2.0 ** -23 * (math.sqrt(M / 16) + 16), 2.0 ** -24 * (math.sqrt(M) + 16)
    dw, db = ops.linear_wgrad_ckpt8(dy.cuda(), x8)
    assert dw.shape == (N, K) and dw.dtype == db.dtype == torch.float32
    assert ((db.double() - rb).abs() <= tolb * mb).all()
    assert ((dw.double() - ref).abs() <= tol * mag).all(), ((dw.double() - ref).abs() / mag).max()
    gw, gb = gamma.double().cuda(), beta.double().cuda()
    dw, db = ops.linear_wgrad_ckpt8(dy.cuda(), x8, gamma=gamma.cuda(), beta=beta.cuda())
    ref2, mag2 = ref * gw + rb[:, None] * gb, mag * gw.abs() + mb[:, None] * gb.abs()
    assert ((dw.double() - ref2).abs() <= (tol + 2.0 ** -22) * mag2).all()
    assert ((db.double() - rb).abs() <= tolb * mb).all()


@pytest.mark.parametrize("M,N,K", [(50, 70, 90), (700, 300, 300), (16384, 1024, 1024), (3000, 256, 96)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_small_whole_numbers_are_exact(M, N, K, dt):
    """every product and partial sum is a whole number below 2^24: any mistake of an index shows"""
    from openvis_amd import ops
    x = ((torch.arange(M * K).reshape(M, K) * 7 // 3) % 15 - 7).float()
    dy = ((torch.arange(M * N).reshape(M, N) * 5 // 2) % 13 - 6).to(T[dt])
    x8 = ops.ckpt8_encode(x.cuda())
    assert torch.equal(_value8(x8).float(), x)
    dw, db = ops.linear_wgrad_ckpt8(dy.cuda(), x8)
    assert torch.equal(dw.double(), dy.cuda().double().t() @ x.cuda().double()) and torch.equal(db.double(), dy.cuda().double().sum(0))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_scales_far_apart(dt):
    """rows of 2^-90 to 2^90: each column block on its own scale, tiny blocks beside large ones"""
    from openvis_amd import ops
    M, N, K = 130, 96, 320
    g = torch.Generator().manual_seed(8)
    e = torch.tensor([-90.0, -60, -30, -10, 0, 10, 30, 60, 80, 1]).repeat_interleave(32)
    x = torch.randn(M, K, generator=g) * 2.0 ** e
    dy = torch.randn(M, N, generator=g).to(T[dt])
    x8 = ops.ckpt8_encode(x.cuda())
    v, d = _value8(x8), dy.double()
    dw, _ = ops.linear_wgrad_ckpt8(dy.cuda(), x8)
    assert ((dw.cpu().double() - d.t() @ v).abs() <= 2.0 ** -23 * 20 * (d.abs().t() @ v.abs())).all()
    # rows of one column block whose scales differ by up to 2^60: off by at most 2^-30 of the block's largest value a row
    x = torch.randn(M, K, generator=g) * 2.0 ** torch.linspace(-30, 30, M)[:, None]
    x8 = ops.ckpt8_encode(x.cuda())
    v = _value8(x8)
    dw, _ = ops.linear_wgrad_ckpt8(dy.cuda(), x8)
    low = v.abs().amax() * 2.0 ** -30 * d.abs().sum(0)[:, None]
    assert ((dw.cpu().double() - d.t() @ v).abs() <= 2.0 ** -23 * 20 * (d.abs().t() @ v.abs()) + (low if dt == "f16" else 0)).all()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_small_gradients(dt):
    """dy down to its type's smallest normal numbers"""
    from openvis_amd import ops
    M, N, K = 96, 64, 64
    g = torch.Generator().manual_seed(2)
    dy = (torch.randn(M, N, generator=g) * {"f32": 2.0 ** -60, "f16": 2.0 ** -10, "bf16": 2.0 ** -60}[dt]).to(T[dt])
    x8 = ops.ckpt8_encode(torch.randn(M, K, generator=g).cuda())
    v, d = _value8(x8), dy.double()
    dw, _ = ops.linear_wgrad_ckpt8(dy.cuda(), x8)
    assert ((dw.cpu().double() - d.t() @ v).abs() <= 2.0 ** -23 * 20 * (d.abs().t() @ v.abs())).all()


def test_gradient_is_that_of_differences():
    """dW and db of sum((x W^T + b) dy) against differences: linear in W and b, so a difference is exact up to rounding"""
    from openvis_amd import ops
    M, N, K = 20, 6, 40
    g = torch.Generator().manual_seed(1)
    x8 = ops.ckpt8_encode(torch.randn(M, K, generator=g).cuda())
    v, dy, W, b = _value8(x8), torch.randn(M, N, generator=g), torch.randn(N, K, generator=g).double(), torch.randn(N, generator=g).double()
    gamma, beta = torch.randn(K, generator=g), torch.randn(K, generator=g)
    f = lambda W_, b_: (((v * gamma.double() + beta.double()) @ W_.t() + b_) * dy.double()).sum().item()
    dw, db = ops.linear_wgrad_ckpt8(dy.cuda(), x8, gamma=gamma.cuda(), beta=beta.cuda())
    for n in range(N):
        e = torch.zeros(N, dtype=torch.float64)
        e[n] = 1
        assert abs(f(W, b + e) - f(W, b) - db[n].item()) < 1e-4
        for k in range(0, K, 3):
            e = torch.zeros(N, K, dtype=torch.float64)
            e[n, k] = 1
            assert abs(f(W + e, b) - f(W, b) - dw[n, k].item()) < 1e-4


def test_not_finite_values_stay_in_their_row_and_column():
    from openvis_amd import ops
    for t in T.values():
        x, dy = torch.ones(200, 100), torch.ones(200, 70).to(t)
        x[3, 40], dy[5, 9] = math.nan, math.inf
        dw, db = (u.cpu() for u in ops.linear_wgrad_ckpt8(dy.cuda(), ops.ckpt8_encode(x.cuda())))
        assert torch.isnan(dw[:, 40]).all() and not torch.isfinite(dw[9]).any() and db[9] == math.inf
        keep_n, keep_k = [n for n in range(70) if n != 9], [k for k in range(100) if k != 40]
        assert (dw[keep_n][:, keep_k] == 200).all() and (db[keep_n] == 200).all()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_strided_rows_no_rows(dt):
    from openvis_amd import ops
    g = torch.Generator().manual_seed(6)
    big = torch.randn(333, 301, generator=g).to(T[dt]).cuda()
    x8 = ops.ckpt8_encode(torch.randn(333, 200, generator=g).cuda())
    v = big[:, 7:140]
    a, b = ops.linear_wgrad_ckpt8(v, x8), ops.linear_wgrad_ckpt8(v.contiguous(), x8)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    dw, db = ops.linear_wgrad_ckpt8(big[:0, :5], ops.ckpt8_encode(torch.empty(0, 40).cuda()))
    assert dw.shape == (5, 40) and not dw.any() and not db.any()


@pytest.mark.parametrize("M,N,K", [(9000, 300, 520), (9000, 2048, 2100)])       # the second: the largest tile, the scales' maxima beforehand
def test_same_bits_on_another_stream_and_in_a_replayed_graph(M, N, K):
    from openvis_amd import ops
    g = torch.Generator().manual_seed(1)
    dy = torch.randn(M, N, generator=g).half().cuda()
    x8 = ops.ckpt8_encode(torch.randn(M, K, generator=g).cuda())
    gamma, beta = torch.randn(K, generator=g).cuda(), torch.randn(K, generator=g).cuda()

    def step():
        return ops.linear_wgrad_ckpt8(dy, x8, gamma=gamma, beta=beta)
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
        dy.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step(), out)), k


def test_refusals():
    from openvis_amd import ops
    from openvis_amd._lib import OvisError
    d, x8, g = torch.zeros(8, 16).cuda(), ops.ckpt8_encode(torch.zeros(8, 64).cuda()), torch.ones(64).cuda()
    bad = [lambda: ops.linear_wgrad_ckpt8(d.double(), x8), lambda: ops.linear_wgrad_ckpt8(d[:7], x8), lambda: ops.linear_wgrad_ckpt8(d.t(), x8),
           lambda: ops.linear_wgrad_ckpt8(d, x8, gamma=g), lambda: ops.linear_wgrad_ckpt8(d, x8, gamma=g[:32], beta=g), lambda: ops.linear_wgrad_ckpt8(d.cpu(), x8),
           lambda: ops.linear_wgrad_ckpt8(d, x8, gamma=g.half(), beta=g.half()), lambda: ops.linear_wgrad_ckpt8(d, (x8.codes, g)),
           lambda: ops.linear_wgrad_ckpt8(d[:, :0], x8)]
    for f in bad:
        with pytest.raises(OvisError):
            f()
