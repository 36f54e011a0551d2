"""GPU: the weight gradient from an 8-bit input whose rows are far apart in size, against 64 bits.

Tolerances as in test_wgrad_ckpt8_gpu.py: every product is exact, a matrix instruction adds 16 at a time: 2^-23 * (sqrt(M / 16) + 16) of the sum of
the magnitudes for random terms (in bf16 an fp16 gradient is two terms, twice as many additions)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# one workgroup; the three tile sizes; rows in one part and in several; column counts that end inside a tile and a block
SHAPES = [(40, 70, 90), (700, 300, 300), (3000, 256, 96), (2500, 768, 768), (9000, 1030, 520), (9000, 2048, 2100)]


def _value8(ck):
    C = ck.codes.shape[1]
    return ck.codes.cpu().double() * ck.scales.cpu().double().repeat_interleave(32, 1)[:, :C]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dt", list(T))
def test_large_rows_without_a_gradient_cost_nothing(M, N, K, dt):
    """padding rows hold anything, here values around 2^50, and their gradient is 0: the sums are those of the other rows"""
    from openvis_amd import ops
    g = torch.Generator().manual_seed(M + K)
    x = torch.randn(M, K, generator=g)
    dy = torch.randn(M, N, generator=g).to(T[dt])
    pad = torch.rand(M, generator=g) < 0.1
    pad[M // 2] = True
    x[pad] *= 2.0 ** 50
    dy[pad] = 0
    x8 = ops.ckpt8_encode(x.cuda())
    v, d = _value8(x8).cuda(), dy.double().cuda()
    ref, mag = d.t().contiguous() @ v, d.abs().t().contiguous() @ v.abs()
    dw, db = ops.linear_wgrad_ckpt8(dy.cuda(), x8)
    assert ((dw.double() - ref).abs() <= 2.0 ** -23 * (math.sqrt(M / 8) + 16) * mag).all(), ((dw.double() - ref).abs() / mag).max()
    assert ((db.double() - d.sum(0)).abs() <= 2.0 ** -24 * (math.sqrt(M) + 16) * d.abs().sum(0)).all()
    again, _ = ops.linear_wgrad_ckpt8(dy.cuda(), x8)
    assert torch.equal(dw, again)


@pytest.mark.parametrize("far", [10, 20, 25, 30, 60, 150])
@pytest.mark.parametrize("M,N,K", [(300, 70, 90), (5000, 384, 96)])
def test_whole_numbers_beside_large_rows_are_exact(M, N, K, far):
    """fp16 gradients: whole numbers times 2^-far, a row of ones without a gradient in each 32 columns: every sum is a whole number below 2^24"""
    from openvis_amd import ops
    step = 2.0 ** -min(far, 90)
    x = ((torch.arange(M * K).reshape(M, K) * 7 // 3) % 15 - 7).float() * step
    dy = ((torch.arange(M * N).reshape(M, N) * 5 // 2) % 13 - 6).half()
    x[M // 3], dy[M // 3] = (2.0 ** 60 if far > 90 else 1.0), 0
    x[7, :5], dy[9] = 0, dy[9] * 2.0 ** -4 * 16
    x8 = ops.ckpt8_encode(x.cuda())
    assert torch.equal(_value8(x8).float(), x)
    gamma, beta = torch.full((K,), 2.0).cuda(), torch.full((K,), step).cuda()
    want = dy.double().t() @ x.double()
    dw, db = ops.linear_wgrad_ckpt8(dy.cuda(), x8)
    assert torch.equal(dw.cpu().double(), want) and torch.equal(db.cpu().double(), dy.double().sum(0))
    dw, _ = ops.linear_wgrad_ckpt8(dy.cuda(), x8, gamma=gamma, beta=beta)
    assert torch.equal(dw.cpu().double(), 2 * want + dy.double().sum(0)[:, None] * step)


def test_not_finite_values_beside_large_rows():
    from openvis_amd import ops
    x, dy = torch.full((200, 100), 2.0 ** -30), torch.ones(200, 70).half()
    x[0], dy[0] = 1.0, 0
    x[3, 40], dy[5, 9], dy[6, 10] = math.nan, math.inf, -math.inf
    dw, db = (u.cpu() for u in ops.linear_wgrad_ckpt8(dy.cuda(), ops.ckpt8_encode(x.cuda())))
    keep_n, keep_k = [n for n in range(70) if n not in (9, 10)], [k for k in range(100) if k != 40]
    assert torch.isnan(dw[:, 40]).all() and (dw[9, keep_k] == math.inf).all() and (dw[10, keep_k] == -math.inf).all()
    assert (dw[keep_n][:, keep_k] == 199 * 2.0 ** -30).all() and (db[keep_n] == 199).all()


def test_blocks_of_the_smallest_scale():
    """zeros have the scale 2^-100 and cost nothing; values that need it count beside scales below 2^-77, and are at most 2^-91 where they do not"""
    from openvis_amd import ops
    M, N, K = 200, 70, 90
    x = ((torch.arange(M * K).reshape(M, K) * 7 // 3) % 15 - 7).float()
    dy = ((torch.arange(M * N).reshape(M, N) * 5 // 2) % 13 - 6).half()
    for large in (2.0 ** -69, 1.0):                              # 7 * 2^-78: its scale is 2^-83; 7 * 2^-9: 2^-14
        y = x * torch.where(torch.arange(M) % 2 == 0, 2.0 ** -96, large * 2.0 ** -9)[:, None]
        y[5:20] = 0
        x8 = ops.ckpt8_encode(y.cuda())
        assert torch.equal(_value8(x8).float(), y)
        dw, _ = ops.linear_wgrad_ckpt8(dy.cuda(), x8)
        want = dy.double().t() @ y.double()
        # the sums' terms are whole numbers of one size, and of another 2^18 or 2^87 below: a rounding of 2^-23 each M / 16 times
        room = 2.0 ** -23 * (math.sqrt(M / 16) + 16) * (dy.double().abs().t() @ y.double().abs())
        if large == 1.0:
            room = room + dy.double().abs().sum(0)[:, None] * 2.0 ** -91
        assert ((dw.cpu().double() - want).abs() <= room).all()
    y = x * 2.0 ** -96                                           # all of them: exact
    dw, _ = ops.linear_wgrad_ckpt8(dy.cuda(), ops.ckpt8_encode(y.cuda()))
    assert torch.equal(dw.cpu().double(), dy.double().t() @ y.double())
