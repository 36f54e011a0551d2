"""GPU: the weight gradient from an 8-bit input at the ends of dy's range, and over long sums of one sign, against 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _value8(ck):
    C = ck.codes.shape[1]
    return ck.codes.double() * ck.scales.double().repeat_interleave(32, 1)[:, :C]


@pytest.mark.parametrize("M,N,K", [(20, 70, 90), (600, 200, 300)])
@pytest.mark.parametrize("dt", list(T))
def test_the_largest_gradients(M, N, K, dt):
    """dy up to its type's largest value; x of at most 2^-40 keeps the sums finite.  Every product is exact: a rounding of 2^-23 each 16 rows, of
    three terms for f32"""
    from openvis_amd import ops
    g = torch.Generator().manual_seed(M)
    top = torch.finfo(T[dt]).max
    dy = torch.where(torch.rand(M, N, generator=g) < 0.5, 1.0, -1.0).double() * top * (1 - 2.0 ** -4 * torch.rand(M, N, generator=g))
    dy[::3] = top
    dy = dy.to(T[dt])
    assert torch.isfinite(dy).all() and dy.max() == top
    x8 = ops.ckpt8_encode((torch.randn(M, K, generator=g) * 2.0 ** -43).cuda())
    dw, _ = ops.linear_wgrad_ckpt8(dy.cuda(), x8)
    v, d = _value8(x8).cpu(), dy.double()
    assert ((dw.cpu().double() - d.t() @ v).abs() <= 2.0 ** -23 * (math.sqrt(3 * M / 16) + 16) * (d.abs().t() @ v.abs())).all()


@pytest.mark.parametrize("dt,exps", [("f32", (-149, -140, -133, -126, -118, -111, -100)), ("bf16", (-133, -130, -126, -120)), ("f16", (-24, -20, -14))])
def test_the_smallest_gradients(dt, exps):
    """dy down to its type's last bit.  f32 is exact from 2^-110 on; below, what three bf16 numbers do not hold, at most 2^-133 a value, is lost"""
    from openvis_amd import ops
    M, N, K = 96, 64, 64
    for e in exps:
        g = torch.Generator().manual_seed(-e)
        dy = (torch.randn(M, N, generator=g).double() * 2.0 ** e).to(T[dt])
        x8 = ops.ckpt8_encode((torch.randn(M, K, generator=g) * 2.0 ** 40).cuda())          # the products stay in f32's normal range
        v, d = _value8(x8).cpu(), dy.double()
        dw, db = ops.linear_wgrad_ckpt8(dy.cuda(), x8)
        room = 2.0 ** -23 * 20 * (d.abs().t() @ v.abs()) + (2.0 ** -133 * v.abs().sum(0) if dt == "f32" and e < -108 else 0)
        assert ((dw.cpu().double() - d.t() @ v).abs() <= room).all(), e
        assert ((db.cpu().double() - d.sum(0)).abs() <= 2.0 ** -24 * 26 * d.abs().sum(0) + 2.0 ** -149).all(), e


def test_nan_and_infinities_spoil_their_columns_alone():
    from openvis_amd import ops
    for t in T.values():
        x, dy = torch.ones(200, 100), torch.ones(200, 70).to(t)
        dy[5, 9], dy[6, 10], dy[7, 11] = math.inf, -math.inf, math.nan
        if t == torch.float32:
            dy[8, 12] = torch.tensor(0x7f800001, dtype=torch.int32).view(torch.float32)     # a NaN whose bits lie in the lower half
        dw, db = (u.cpu() for u in ops.linear_wgrad_ckpt8(dy.cuda(), ops.ckpt8_encode(x.cuda())))
        bad = [9, 10, 11] + ([12] if t == torch.float32 else [])
        keep = [n for n in range(70) if n not in bad]
        assert not torch.isfinite(dw[bad]).any() and torch.isnan(dw[bad[2:]]).all() and (dw[keep] == 200).all()
        assert db[9] == math.inf and db[10] == -math.inf and torch.isnan(db[bad[2:]]).all() and (db[keep] == 200).all()


@pytest.mark.parametrize("dt", list(T))
def test_long_sums_of_one_sign_do_not_drift(dt):
    """4096 x 4096 tiles fill the card, so the 36928 rows are one chain of M / 16 additions (three a row of f32).  Rounded to nearest, their errors of
    2^-24 of the sum at most grow with the chain's root: 4 of that for the largest of 2048 sums.  Cut off instead, they would come to 1.4e-4."""
    from openvis_amd import ops
    M = 36928
    g = torch.Generator(device="cuda").manual_seed(1)
    x8 = ops.ckpt8_encode(torch.rand(M, 4096, generator=g, device="cuda"))
    dy = torch.rand(M, 4096, generator=g, device="cuda").to(T[dt])
    dw, db = ops.linear_wgrad_ckpt8(dy, x8)
    v = _value8(ops.Ckpt8(x8.codes[:, :32].contiguous(), x8.scales[:, :1].contiguous()))
    ref = dy[:, :64].double().t().contiguous() @ v
    chain = M / 16 * (3 if dt == "f32" else 1)
    assert ((dw[:64, :32].double() - ref).abs() <= 2.0 ** -24 * (4 * math.sqrt(chain) + 16) * ref).all()
    assert ((db.double() - dy.double().sum(0)).abs() <= 2.0 ** -24 * (math.sqrt(M) + 16) * dy.double().sum(0)).all()
