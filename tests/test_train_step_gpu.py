"""GPU: the training-side operators together, as a fine-tuning step uses them: the MLP half of a transformer block (layer norm -> fc1 ->
activation -> fc2, with the residual) forward and backward on the framework's GEMMs, every intermediate kept in 8 bits, and an attention
whose bias table learns.

What 8 bits cost is part of the operators' definition, so the gradients are checked twice: exactly (to f32 rounding) against the same formulas in
64 bits fed with the values that the 8-bit forms stand for, and loosely against autograd on the un-quantised block, where a code is off by 2^-4
of a value at most and by 2^-4 / sqrt(3) in the mean square: sums of many independent errors stay within 5 % in the 2-norm."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _value8(ck):
    C = ck.codes.shape[1]
    return ck.codes.double() * ck.scales.double().repeat_interleave(32, 1)[:, :C]


def _act64(h, act):
    from openvis_amd import ops
    if act == ops.ACT_RELU:
        return h.clamp(min=0)
    return h * torch.sigmoid(1.702 * h) if act == ops.ACT_QUICKGELU else 0.5 * h * torch.special.erfc(-h / math.sqrt(2))


def _rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("rows,C,F", [(300, 96, 384), (77 * 5, 512, 2048), (1001, 100, 200)])
@pytest.mark.parametrize("act", [1, 2, 3])
def test_mlp_half_block(rows, C, F, act):
    from openvis_amd import ops
    g = torch.Generator().manual_seed(rows + act)
    rnd = lambda *s: torch.randn(*s, generator=g).cuda()
    x, r, dout = rnd(rows, C), rnd(rows, C), rnd(rows, C)
    gamma, beta = 1 + 0.2 * rnd(C), 0.2 * rnd(C)
    w1, b1, w2, b2 = rnd(F, C) / C ** 0.5, 0.1 * rnd(F), rnd(C, F) / F ** 0.5, 0.1 * rnd(C)
    # forward: s = x + r; out = s + fc2(act(fc1(LN(s))))
    ln = ops.layernorm_forward(x, gamma, beta, residual=r, checkpoint=True)
    h = ops.gemm_nt(ln.y, w1, b1)
    a, h8 = ops.act_forward_ckpt8(h, act)
    out = ops.gemm_nt(a, w2, b2, residual=ln.sum)
    # backward: kept are ln.xhat8, ln.stats and h8 alone
    da = ops.gemm_nt(dout, w2.t().contiguous())
    dh, db1, a8 = ops.act_backward_ckpt8(da, h8, act, recompute=True)
    dw2, db2 = ops.linear_wgrad_ckpt8(dout, a8)
    dw1, db1b = ops.linear_wgrad_ckpt8(dh, ln.xhat8, gamma=gamma, beta=beta)
    du = ops.gemm_nt(dh, w1.t().contiguous())
    ds, dgamma, dbeta = ops.layernorm_backward(du, ln.xhat8, ln.stats, gamma, dsum=dout)
    # (1) the same formulas in 64 bits, on the values that the codes stand for
    d = lambda t: t.double()
    xh, hv, av = _value8(ln.xhat8), _value8(h8), _value8(a8)
    hq = hv.clone().requires_grad_()
    if act == 1:
        slope = (~torch.signbit(hv)).double()
    else:
        slope, = torch.autograd.grad(_act64(hq, act).sum(), hq)
    da64 = d(dout) @ d(w2)
    dh64 = da64 * slope
    want = {"dw2": d(dout).t() @ av, "db2": d(dout).sum(0), "db1": dh64.sum(0), "dw1": dh64.t() @ (xh * d(gamma) + d(beta))}
    du64 = dh64 @ d(w1)
    gd, rstd = du64 * d(gamma), d(ln.stats[:, 1:])
    want.update(ds=rstd * (gd - gd.mean(1, keepdim=True) - xh * (gd * xh).mean(1, keepdim=True)) + d(dout), dgamma=(du64 * xh).sum(0), dbeta=du64.sum(0))
    got = dict(dw2=dw2, db2=db2, db1=db1, dw1=dw1, ds=ds, dgamma=dgamma, dbeta=dbeta)
    for k in want:                                   # chains of up to three f32 products of at most 2048 terms: 2^-24 * sqrt(2048) * a few
        assert _rel(got[k], want[k]) < 2.0 ** -24 * 200, (k, _rel(got[k], want[k]))
    assert _rel(db1b, d(dh).sum(0)) < 2.0 ** -24 * 100
    # (2) autograd on the block itself
    P = [t.double().requires_grad_() for t in (x, r, gamma, beta, w1, b1, w2, b2)]
    X, R, Ga, Be, W1, B1, W2, B2 = P
    S = X + R
    ref = S + _act64(torch.nn.functional.layer_norm(S, (C,), Ga, Be, 1e-5) @ W1.t() + B1, act) @ W2.t() + B2
    assert _rel(out, ref.detach()) < 2.0 ** -24 * 200
    ref.backward(d(dout))
    for k, p in (("ds", X), ("ds", R), ("dgamma", Ga), ("dbeta", Be), ("dw1", W1), ("db1", B1), ("dw2", W2), ("db2", B2)):
        assert _rel(got[k], p.grad) < 0.05, (k, _rel(got[k], p.grad))


def test_attention_whose_bias_table_learns():
    """forward on ops.attention with relpos_bias_1d, the scores' gradient by formula, the table's by relpos_bias_1d_backward, against autograd"""
    from openvis_amd import ops
    B, H, N, D, NB = 3, 4, 50, 32, 16
    g = torch.Generator().manual_seed(2)
    q, k, v, do = (torch.randn(B, N, H * D, generator=g).cuda() for _ in range(4))
    table = torch.randn(NB, H, generator=g).cuda()
    ld, s = 52, H * D
    bias = ops.relpos_bias_1d(table, N, N, max_distance=64, ld=ld)
    out = ops.attention(q, k, v, B, H, N, N, D, N * s, s, N * s, s, N * s, s, bias=bias[None], bias_strides=(0, N * ld))
    heads = lambda t: t.double().view(B, N, H, D).transpose(1, 2).contiguous()
    Q, K, V, DO = heads(q), heads(k), heads(v), heads(do)
    T = table.double().requires_grad_()
    e = NB // 4
    bucket = torch.zeros(N, N, dtype=torch.long)
    for i in range(N):
        for j in range(N):
            n = abs(j - i)
            b = n if n < e else max(kk for kk in range(e, NB // 2) if n ** (NB // 2 - e) * e ** (kk - e) >= 64 ** (kk - e) * e ** (NB // 2 - e))
            bucket[i, j] = b + (NB // 2 if j > i else 0)
    sc = Q @ K.transpose(2, 3).contiguous() / math.sqrt(D) + T.t()[:, bucket.cuda()]
    P = sc.softmax(-1)
    ref = P @ V
    assert (heads(out) - ref).abs().max() < 400 * 2.0 ** -24            # scores of magnitude 20 in f32
    (ref * DO).sum().backward()
    with torch.no_grad():
        dp = DO @ V.transpose(2, 3).contiguous()
        dS = P * (dp - (dp * P).sum(-1, keepdim=True))
    got = ops.relpos_bias_1d_backward(dS.float(), NB, max_distance=64)
    assert _rel(got, T.grad) < 2.0 ** -24 * 50


def test_two_graphs_share_no_workspace():
    """two captured steps of different sizes, replayed in turn with eager calls between: every replay as the eager call"""
    from openvis_amd import ops
    g = torch.Generator().manual_seed(5)
    sets = []
    for rows, C in ((2000, 256), (513, 1000)):
        x, dy = torch.randn(rows, C, generator=g).half().cuda(), torch.randn(rows, C, generator=g).half().cuda()
        gamma, beta = torch.randn(C, generator=g).cuda(), torch.randn(C, generator=g).cuda()

        def step(x=x, dy=dy, gamma=gamma, beta=beta):
            o = ops.layernorm_forward(x, gamma, beta, checkpoint=True)
            y, h8 = ops.act_forward_ckpt8(o.y, ops.ACT_GELU)
            dh, db, a8 = ops.act_backward_ckpt8(dy, h8, ops.ACT_GELU, recompute=True)
            return (y, dh, db) + ops.linear_wgrad_ckpt8(dy, a8) + ops.layernorm_backward(dh, o.xhat8, o.stats, gamma, dsum=dy)
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        sets.append((x, step, graph, out))
    for k in range(3):
        for x, _, _, _ in sets:
            x.mul_(0.9)
        for _, _, graph, _ in sets:
            graph.replay()
        torch.cuda.synchronize()
        for _, step, _, out in sets:
            assert all(torch.equal(a, b) for a, b in zip(step(), out)), k
