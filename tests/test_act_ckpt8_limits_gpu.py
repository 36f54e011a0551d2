"""GPU: the activations that are kept in 8 bits at the ends of their types' ranges."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dt", list(T))
@pytest.mark.parametrize("C", [5, 32, 100])
def test_relu_of_infinities(dt, C):
    """-infinity (an fp16 layer that overflowed) is a value below 0: activation 0, slope 0, and nothing of it in the sums or in the activation
    that is computed again; +infinity and NaN stay what they are"""
    from openvis_amd import ops
    g = torch.Generator().manual_seed(C)
    h = torch.randn(7, C, generator=g)
    low = torch.rand(7, C, generator=g) < 0.3
    low[2], low[3, :4] = True, True
    low[5, 0] = low[6, 1] = False
    h[low] = -math.inf
    h[5, 0], h[6, 1] = math.inf, math.nan
    dy = torch.randn(7, C, generator=g).to(T[dt])
    y, ck = ops.act_forward_ckpt8(h.to(T[dt]).cuda(), ops.ACT_RELU)
    y, odd = y.cpu(), ~torch.isfinite(h) & ~low
    assert torch.equal(y[~odd], h.to(T[dt]).clamp(min=0)[~odd]) and y[5, 0] == math.inf and torch.isnan(y[6, 1])
    codes = ck.codes.cpu().float()
    assert torch.equal(codes[low], torch.zeros(int(low.sum()))) and torch.signbit(codes[low]).all() and torch.isnan(codes[odd]).all() and not torch.signbit(codes[odd]).any()
    finite = torch.where(low, torch.zeros_like(h), h)             # the other values' codes and scales are those without the infinities
    _, other = ops.act_forward_ckpt8(finite.to(T[dt]).cuda(), ops.ACT_RELU)
    assert torch.equal(ck.codes.view(torch.uint8), other.codes.view(torch.uint8)) and torch.equal(ck.scales.view(torch.uint8), other.scales.view(torch.uint8))
    dh, db, y8 = ops.act_backward_ckpt8(dy.cuda(), ck, ops.ACT_RELU, recompute=True)
    want = torch.where((h > 0) | torch.isnan(h), dy.float(), torch.zeros_like(h))
    assert torch.equal(dh.cpu(), want.to(T[dt]))
    # seven terms: at most six roundings of 2^-24 of the sum of the magnitudes each
    assert ((db.cpu().double() - want.double().sum(0)).abs() <= 6 * 2.0 ** -24 * want.double().abs().sum(0)).all()
    again = y8.codes.cpu().float()
    assert torch.equal(again[low], torch.zeros(int(low.sum()))) and torch.isfinite(again[~odd]).all() and torch.isnan(again[odd]).all()


@pytest.mark.parametrize("act", ["quickgelu", "gelu"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_the_largest_values(act, dt):
    """values up to the 8-bit form's largest, 448 * 2^119: the activation is h or 0 and the slope 1 or 0, exactly, and none of it NaN"""
    from openvis_amd import ops
    code = {"quickgelu": ops.ACT_QUICKGELU, "gelu": ops.ACT_GELU}[act]
    h = torch.tensor([[s * m * 2.0 ** e for m in (1.0, 1.25, 1.75) for s in (1, -1)] for e in (20, 63, 64, 100, 126, 127)])
    y, ck = ops.act_forward_ckpt8(h.to(T[dt]).cuda(), code)
    assert torch.equal(y.cpu().float(), h.clamp(min=0))
    dh, db, y8 = ops.act_backward_ckpt8(torch.ones_like(y), ck, code, recompute=True)
    assert torch.equal(dh.cpu().float(), (h > 0).float()) and torch.equal(db.cpu(), (h > 0).float().sum(0))
    assert torch.equal(ops.ckpt8_decode(y8).cpu(), h.clamp(min=0))
