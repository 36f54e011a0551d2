"""GPU: relative position bias by buckets and the gradients of its tables (csrc/relpos.hip, swin_ops.hip) against plain loops in whole numbers and
64 bits.

Tolerances: the bias is a copy, rounded once: compared for equality.  A gradient is a sum of n terms in f32, taken in parts of at most 64 K
terms one after another and then pairwise: 2^-24 * (sqrt(n) + 16) of the sum of the magnitudes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _buckets(num, dist, both):
    """bucket of a distance 0..: by fractions of whole numbers, no logarithm"""
    n = num // 2 if both else num
    e = n // 2
    first = list(range(e + 1))
    for k in range(1, n - e):
        d = first[-1]
        while d ** (n - e) * e ** k < dist ** k * e ** (n - e):
            d += 1
        first.append(d)
    return lambda d: max(b for b, f in enumerate(first) if d >= f)


def _map(Nq, Nk, num, dist, both, off):
    """bucket of each diagonal j - i = -(Nq - 1) .. Nk - 1, and of each (i, j)"""
    of, n = _buckets(num, dist, both), num // 2 if both else num
    line = [of(abs(r)) + (n if r > 0 else 0) if both else of(max(-r, 0)) for r in range(-(Nq - 1) - off, Nk - off)]
    line = torch.tensor(line)
    return line[torch.arange(Nk)[None, :] - torch.arange(Nq)[:, None] + Nq - 1]


CASES = [(1, 1, 8, 64, True, 0), (1, 1, 32, 128, False, 0), (1, 300, 32, 128, False, 299), (1, 4097, 32, 128, True, 4000), (7, 5, 8, 16, True, 0),
         (64, 64, 32, 128, True, 0), (65, 63, 32, 128, False, -2), (129, 520, 16, 100, False, 391), (200, 200, 64, 1000, True, 3),
         (513, 1025, 32, 128, True, 512), (1030, 70, 32, 128, True, 0), (1, 9, 2, 2, False, 8), (33, 33, 4, 2, True, 0), (70, 2100, 32, 128, False, 2030),
         (5, 40, 32, 128, False, 10 ** 12), (5, 40, 32, 128, True, -10 ** 12)]


@pytest.mark.parametrize("Nq,Nk,num,dist,both,off", CASES)
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_bias_and_gradient_of_sequences(Nq, Nk, num, dist, both, off, dt):
    from openvis_amd import ops
    H, B = 3, 5
    g = torch.Generator().manual_seed(Nq * 7 + Nk)
    table = torch.randn(num, H, generator=g)
    if abs(off) > 10 ** 9:
        n = num // 2 if both else num
        m = torch.full((Nq, Nk), n - 1 if not both or off > 0 else num - 1)
    else:
        m = _map(Nq, Nk, num, dist, both, off)
    bias = ops.relpos_bias_1d(table.cuda(), Nq, Nk, dist, both, off, out_dtype=T[dt])
    assert bias.shape == (H, Nq, Nk) and torch.equal(bias.cpu(), table.t()[:, m].to(T[dt]))
    ld = (Nk + 7) // 8 * 8 + 8
    full = ops.relpos_bias_1d(table.cuda(), Nq, Nk, dist, both, off, out_dtype=T[dt], ld=ld)
    assert full.shape == (H, Nq, ld) and torch.equal(full[..., :Nk].cpu(), bias.cpu()) and not full[..., Nk:].any()
    d = torch.randn(B, H, Nq, Nk, generator=g).to(T[dt])
    for x in (d, d[0]):
        got = ops.relpos_bias_1d_backward(x.cuda(), num, dist, both, off)
        x = (x if x.dim() == 4 else x[None]).double()
        ref, mag, cnt = (torch.zeros(num, H, dtype=torch.float64) for _ in range(3))
        idx = m.reshape(-1)
        ref.index_add_(0, idx, x.sum(0).reshape(H, -1).t())
        mag.index_add_(0, idx, x.abs().sum(0).reshape(H, -1).t())
        cnt.index_add_(0, idx, torch.full((H, idx.numel()), float(x.shape[0]), dtype=torch.float64).t())
        assert got.shape == (num, H) and got.dtype == torch.float32
        assert ((got.cpu().double() - ref).abs() <= 2.0 ** -24 * (cnt.sqrt() + 16) * mag).all()


def _window_index(ws):
    p = torch.arange(ws * ws)
    y, x = p // ws, p % ws
    return (y[:, None] - y[None] + ws - 1) * (2 * ws - 1) + x[:, None] - x[None] + ws - 1


@pytest.mark.parametrize("B,H,ws", [(1, 1, 1), (1, 3, 2), (2, 5, 3), (37, 4, 7), (100, 6, 12), (3, 2, 16), (1, 1, 20), (2111, 1, 4), (5000, 3, 2)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_gradient_of_windows(B, H, ws, dt):
    from openvis_amd import ops
    N, g = ws * ws, torch.Generator().manual_seed(B + ws)
    d = torch.randn(B, H, N, N, generator=g).to(T[dt])
    got = ops.swin_relpos_bias_backward(d.cuda(), ws)
    idx = _window_index(ws).reshape(-1)
    ref, mag = (torch.zeros((2 * ws - 1) ** 2, H, dtype=torch.float64) for _ in range(2))
    ref.index_add_(0, idx, d.double().sum(0).reshape(H, -1).t())
    mag.index_add_(0, idx, d.double().abs().sum(0).reshape(H, -1).t())
    assert got.shape == ref.shape and ((got.cpu().double() - ref).abs() <= 2.0 ** -24 * (math.sqrt(B * N) + 16) * mag).all()
    # the bias whose table's gradient this is: <bias(t), sum d> = <t, grad> for every table t
    table = torch.randn((2 * ws - 1) ** 2, H, generator=g)
    bias = ops.swin_relpos_bias(table.cuda(), H, ws, (N + 3) // 4 * 4)[..., :N].cpu().double()
    lhs, rhs = (bias * d.double().sum(0)).sum(), (table.double() * got.cpu().double()).sum()
    assert abs(lhs - rhs) <= 2.0 ** -24 * (math.sqrt(B * N) + 16) * (table.double().abs() * mag).sum() + 1e-12


def test_padding_and_strides_are_not_read():
    """padded columns hold NaN; a batch and heads that are far apart, a broadcast batch"""
    from openvis_amd import ops
    g = torch.Generator().manual_seed(0)
    for dt in T.values():
        big = torch.full((3, 4, 50, 71), math.nan, dtype=dt)
        big[:, :, :49, 3:52] = torch.randn(3, 4, 49, 49, generator=g).to(dt)
        big = big.cuda()
        v = big[:, 1:4, :49, 3:52]
        assert torch.equal(ops.swin_relpos_bias_backward(v, 7), ops.swin_relpos_bias_backward(v.contiguous(), 7))
        assert torch.equal(ops.relpos_bias_1d_backward(v, 32), ops.relpos_bias_1d_backward(v.contiguous(), 32))
        pad = torch.full((2, 3, 49, 52), math.nan, dtype=dt).cuda()
        pad[..., :49] = v[:2]
        assert torch.equal(ops.swin_relpos_bias_backward(pad, 7), ops.swin_relpos_bias_backward(v[:2].contiguous(), 7))
        e = v[:1].expand(6, 3, 49, 49)
        assert torch.equal(ops.swin_relpos_bias_backward(e, 7), ops.swin_relpos_bias_backward(e.contiguous(), 7))
        t = v.transpose(0, 1)                                     # batch and heads swapped
        assert torch.equal(ops.relpos_bias_1d_backward(t, 8, 64, False), ops.relpos_bias_1d_backward(t.contiguous(), 8, 64, False))


def test_not_finite_gradients_stay_in_their_bucket():
    from openvis_amd import ops
    d = torch.zeros(1, 1, 40, 600)
    d[0, 0, 7, 6], d[0, 0, 3, 500] = math.nan, math.inf           # distances -1 and 497
    got = ops.relpos_bias_1d_backward(d.cuda(), 32).cpu()[:, 0]
    assert torch.isnan(got[1]) and got[31] == math.inf and torch.isfinite(got[[k for k in range(32) if k not in (1, 31)]]).all()


def test_empty_batches_and_lengths():
    from openvis_amd import ops
    t = torch.randn(32, 2).cuda()
    assert ops.relpos_bias_1d(t, 0, 5).shape == (2, 0, 5) and ops.relpos_bias_1d(t, 5, 0).shape == (2, 5, 0)
    assert not ops.relpos_bias_1d(t, 3, 0, ld=8).any()
    assert not ops.relpos_bias_1d_backward(torch.empty(0, 2, 5, 5).cuda(), 32).any()
    assert not ops.relpos_bias_1d_backward(torch.empty(3, 2, 5, 0).cuda(), 32).any()
    assert ops.swin_relpos_bias_backward(torch.empty(0, 2, 49, 49).cuda(), 7).shape == (169, 2)


def test_with_attention_and_one_new_token():
    """the bias under the framework's attention, a whole causal sequence and its last token alone: the same row"""
    from openvis_amd import ops
    H, N, D = 4, 77, 32
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(1, N, H * D, generator=g).cuda() for _ in range(3))
    table = torch.randn(32, H, generator=g).cuda()
    ld = 80
    bias = ops.relpos_bias_1d(table, N, N, bidirectional=False, ld=ld)
    mask = torch.zeros(N, ld, dtype=torch.uint8)
    mask[:, :N] = torch.triu(torch.ones(N, N), 1)
    s = H * D
    out = ops.attention(q, k, v, 1, H, N, N, D, N * s, s, N * s, s, N * s, s, mask=mask.cuda(), bias=bias[None], bias_strides=(0, N * ld))
    qq, kk, vv = (t.double().cpu().view(N, H, D).transpose(0, 1) for t in (q, k, v))
    score = qq @ kk.transpose(1, 2) / math.sqrt(D) + bias[..., :N].cpu().double()
    ref = score.masked_fill(torch.triu(torch.ones(N, N, dtype=torch.bool), 1), -math.inf).softmax(-1) @ vv
    # scores of magnitude 20 in f32: a relative 20 * 2^-24 * a few on the probabilities
    assert (out.view(N, H, D).transpose(0, 1).cpu().double() - ref).abs().max() < 400 * 2.0 ** -24
    row = ops.relpos_bias_1d(table, 1, N, bidirectional=False, q_offset=N - 1, ld=ld)
    assert torch.equal(row[:, 0], bias[:, N - 1])
    one = ops.attention(q[:, -1:].contiguous(), k, v, 1, H, 1, N, D, s, s, N * s, s, N * s, s, bias=row[None], bias_strides=(0, ld))
    assert (one.view(H, D).cpu().double() - ref[:, -1]).abs().max() < 400 * 2.0 ** -24


def test_same_bits_on_another_stream_and_in_a_replayed_graph():
    from openvis_amd import ops
    g = torch.Generator().manual_seed(1)
    table = torch.randn(32, 6, generator=g).cuda()
    d, w = torch.randn(9, 6, 301, 500, generator=g).half().cuda(), torch.randn(200, 6, 49, 49, generator=g).cuda()

    def step():
        return ops.relpos_bias_1d(table, 301, 500), ops.relpos_bias_1d_backward(d, 32), ops.swin_relpos_bias_backward(w, 7)
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
        table.mul_(1.5), d.mul_(0.5), w.mul_(-2)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step(), out)), k


def test_refusals():
    from openvis_amd import ops
    from openvis_amd._lib import OvisError
    t, d = torch.zeros(32, 2).cuda(), torch.zeros(1, 2, 49, 49).cuda()
    bad = [lambda: ops.relpos_bias_1d(t.half(), 4, 4), lambda: ops.relpos_bias_1d(t.cpu(), 4, 4), lambda: ops.relpos_bias_1d(t[:31], 4, 4),
           lambda: ops.relpos_bias_1d(t, 4, 4, max_distance=8), lambda: ops.relpos_bias_1d(t, 4, 4, ld=3), lambda: ops.relpos_bias_1d(t, 4, 4, ld=6),
           lambda: ops.relpos_bias_1d(t, -1, 4), lambda: ops.relpos_bias_1d(t, 4, 4, out_dtype=torch.float64), lambda: ops.relpos_bias_1d(t.t(), 4, 4),
           lambda: ops.relpos_bias_1d(torch.zeros(1, 2).cuda(), 4, 4, bidirectional=False),
           lambda: ops.relpos_bias_1d_backward(d.double(), 32), lambda: ops.relpos_bias_1d_backward(d[0, 0], 32), lambda: ops.relpos_bias_1d_backward(d, 3),
           lambda: ops.relpos_bias_1d_backward(d.transpose(2, 3)[..., :7], 32), lambda: ops.relpos_bias_1d_backward(d.cpu(), 32),
           lambda: ops.swin_relpos_bias_backward(d, 6), lambda: ops.swin_relpos_bias_backward(d[..., :48], 7), lambda: ops.swin_relpos_bias_backward(d, 65)]
    for f in bad:
        with pytest.raises(OvisError):
            f()
