"""CPU: what the training-side operators check before any device work, the shapes they give, and the bucket borders."""
import ctypes
import math
import re

import pytest
import torch

from openvis_amd import _lib, ops


def _prototypes():
    src = re.sub(r"/\*.*?\*/", "", open(_lib.HEADER_PATH).read(), flags=re.S)
    out = {}
    for ret, name, args in re.findall(r"\b(int|long long|const char\*)\s+(ovis_[a-z0-9_]+)\s*\(([^)]*)\)", src):
        sig = ""
        for a in args.split(","):
            a = a.strip()
            sig += "" if a in ("void", "") else "p" if "*" in a or "ovis_stream_t" in a else "l" if "long long" in a or "int64_t" in a else "f" if a.startswith("float") else "i"
        out[name] = ({"int": "i", "long long": "l"}.get(ret, "s"), sig)
    return out


def _entry(name, signature, returns="i"):
    """the C function with the argument types of its prototype in the header"""
    assert _prototypes()[name] == (returns, signature), name
    t = {"p": ctypes.c_void_p, "i": ctypes.c_int, "l": ctypes.c_longlong, "f": ctypes.c_float}
    return ctypes.CFUNCTYPE(t[returns], *[t[c] for c in signature])((name, _lib.lib()))


def _refused(name, sig, *args):
    if torch.cuda.is_available():
        pytest.skip("the pointers are none: a call that is not refused must find no device")
    rc = _entry(name, sig)(*args)
    assert rc == 1, (name, rc)
    return _lib.lib().ovis_last_error().decode()


P = 1 << 20            # a pointer that is never followed: every call below is refused on the host


def test_layernorm_entry_points_refuse():
    fwd = lambda **k: _refused("ovis_layernorm_train_forward", "plplppppppplifiip", *[{**dict(x=P, ldx=64, res=None, ldr=0, g=P, b=P, sum=None, y=P, st=P,
                               co=None, sc=None, rows=4, C=64, eps=1e-5, xt=0, yt=0, s=None), **k}[n] for n in
                               ("x", "ldx", "res", "ldr", "g", "b", "sum", "y", "st", "co", "sc", "rows", "C", "eps", "xt", "yt", "s")])
    assert "null" in fwd(x=None) and "null" in fwd(res=P, ldr=64) and "null" in fwd(co=P)
    assert "columns" in fwd(C=0) and "columns" in fwd(C=8193, ldx=9000) and "columns" in fwd(rows=0)
    assert "stride" in fwd(ldx=63) and "stride" in fwd(res=P, sum=P, ldr=8)
    assert "type" in fwd(xt=1, yt=0) and "type" in fwd(xt=3, yt=3) and "type" in fwd(yt=-1)
    bwd = lambda **k: _refused("ovis_layernorm_train_backward", "plplppppplppppliiip", *[{**dict(dy=P, ldd=64, x=P, ldx=64, co=None, sc=None, st=P, g=P, ds=None,
                               lds=0, dx=P, dg=P, db=P, ws=P, rows=4, C=64, yt=0, xt=0, s=None), **k}[n] for n in
                               ("dy", "ldd", "x", "ldx", "co", "sc", "st", "g", "ds", "lds", "dx", "dg", "db", "ws", "rows", "C", "yt", "xt", "s")])
    assert "exactly one" in bwd(x=None) and "exactly one" in bwd(co=P, sc=P) and "null" in bwd(ws=None) and "null" in bwd(sc=P)
    assert "stride" in bwd(ldd=3) and "stride" in bwd(ds=P, lds=1) and "type" in bwd(xt=1, yt=2) and "columns" in bwd(rows=-1)
    assert _entry("ovis_layernorm_train_backward_workspace_bytes", "lii", "l")(0, 64, 0) == 0


def test_activation_and_8_bit_entry_points_refuse():
    fwd = lambda *a: _refused("ovis_act_ckpt8_forward", "plpppliiip", *a)
    assert "null" in fwd(None, 64, P, P, P, 4, 64, 3, 0, None) and "null" in fwd(P, 64, None, P, P, 4, 64, 3, 0, None) and "null" in fwd(P, 64, P, P, P, 4, 64, 0, 0, None)
    assert "activation" in fwd(P, 64, P, P, P, 4, 64, 4, 0, None) and "type" in fwd(P, 64, P, P, P, 4, 64, 3, 7, None)
    assert "stride" in fwd(P, 63, P, P, P, 4, 64, 3, 0, None) and "rows" in fwd(P, 64, P, P, P, 0, 64, 3, 0, None)
    assert "too large" in fwd(P, 64, P, P, P, 1 << 40, 64, 3, 0, None)
    bwd = lambda *a: _refused("ovis_act_ckpt8_backward", "plpppppppliiip", *a)
    assert "null" in bwd(P, 64, P, P, P, None, None, None, P, 4, 64, 3, 0, None) and "null" in bwd(P, 64, P, P, P, P, P, None, P, 4, 64, 3, 0, None)
    assert "activation" in bwd(P, 64, P, P, P, P, None, None, P, 4, 64, 0, 0, None) and "stride" in bwd(P, 8, P, P, P, P, None, None, P, 4, 64, 1, 0, None)
    dec = lambda *a: _refused("ovis_ckpt8_decode", "pppliip", *a)
    assert "null" in dec(P, None, P, 4, 64, 0, None) and "type" in dec(P, P, P, 4, 64, 5, None) and "too large" in dec(P, P, P, 1 << 40, 64, 0, None)


def test_relative_position_entry_points_refuse():
    b = (ctypes.c_int * 3)(1, 2, 4)
    fwd = lambda *a: _refused("ovis_relpos_bias_1d", "pppiiiiiilip", *a)
    assert "null" in fwd(None, P, b, 3, 1, 2, 4, 4, 4, 0, 0, None) and "Nq 0" in fwd(P, P, b, 3, 1, 2, 0, 4, 4, 0, 0, None)
    assert "16-byte" in fwd(P, P, b, 3, 1, 2, 4, 5, 5, 0, 0, None) and "16-byte" in fwd(P, P + 4, b, 3, 1, 2, 4, 4, 4, 0, 0, None)
    assert "16-byte" in fwd(P, P, b, 3, 1, 2, 4, 4, 4, 0, 1, None)                      # eight fp16 elements
    assert "ascending" in fwd(P, P, (ctypes.c_int * 3)(1, 4, 2), 3, 1, 2, 4, 4, 4, 0, 0, None) and "ascending" in fwd(P, P, (ctypes.c_int * 1)(0), 1, 1, 2, 4, 4, 4, 0, 0, None)
    assert "borders" in fwd(P, P, b, 257, 1, 2, 4, 4, 4, 0, 0, None) and "borders" in fwd(P, P, None, 3, 1, 2, 4, 4, 4, 0, 0, None)
    bwd = lambda *a: _refused("ovis_relpos_bias_1d_backward", "plllpppiiliiilip", *a)
    assert "null" in bwd(P, 16, 16, 4, P, None, b, 3, 1, 1, 2, 4, 4, 0, 0, None) and "negative" in bwd(P, -1, 16, 4, P, P, b, 3, 1, 1, 2, 4, 4, 0, 0, None)
    assert "B 0" in bwd(P, 16, 16, 4, P, P, b, 3, 1, 0, 2, 4, 4, 0, 0, None) and "too large" in bwd(P, 16, 16, 4, P, P, b, 3, 1, 1, 60000, 1 << 20, 4, 0, 0, None)
    win = lambda *a: _refused("ovis_swin_relpos_bias_backward", "plllppliiip", *a)
    assert "window" in win(P, 0, 0, 0, P, P, 1, 2, 65, 0, None) and "null" in win(P, 0, 0, 0, None, P, 1, 2, 7, 0, None)
    assert "too large" in win(P, 0, 0, 0, P, P, 1, 200, 64, 0, None)


def test_weight_gradient_entry_point_refuses():
    f = lambda *a: _refused("ovis_linear_wgrad_ckpt8", "plpppppppliiip", *a)
    ok = [P, 64, P, P, None, None, P, P, P, 100, 64, 64, 1, None]
    change = lambda **k: f(*[k.get("a%d" % i, v) for i, v in enumerate(ok)])
    assert "null" in change(a0=None) and "null" in change(a4=P) and "null" in change(a8=None)
    assert "stride" in change(a1=63) and "M 0" in change(a9=0) and "type" in change(a12=9)
    assert "too large" in change(a1=1 << 24) and "too large" in change(a11=1 << 24)


def test_launches_of_2_to_the_32_lanes_are_refused():
    """all of these fit in the card's memory, but not in one launch"""
    assert "too many for one launch" in _refused("ovis_layernorm_train_forward", "plplppppppplifiip", P, 8, None, 0, P, P, None, P, P, None, None, 1 << 28, 8,
                                                 1e-5, 1, 1, None)
    b = (ctypes.c_int * 3)(1, 2, 4)
    assert "too large" in _refused("ovis_relpos_bias_1d_backward", "plllpppiiliiilip", P, 0, 0, 1, P, P, b, 3, 1, 1, 1, (1 << 30) - 1, 66, 0, 1, None)
    assert "too large" in _refused("ovis_linear_wgrad_ckpt8", "plpppppppliiip", P, 1 << 20, P, P, None, None, P, P, P, 1, 1 << 20, 1 << 20, 1, None)


def test_tensors_on_the_host_are_refused():
    x, g = torch.zeros(4, 64), torch.ones(64)
    ck = ops.Ckpt8(torch.zeros(4, 64).to(torch.float8_e4m3fn), torch.zeros(4, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu))
    for f in (lambda: ops.layernorm_forward(x, g, g), lambda: ops.layernorm_backward(x, x, torch.zeros(4, 2), g), lambda: ops.ckpt8_encode(x),
              lambda: ops.ckpt8_decode(ck), lambda: ops.act_forward_ckpt8(x, 3), lambda: ops.act_backward_ckpt8(x, ck, 3), lambda: ops.linear_wgrad_ckpt8(x, ck),
              lambda: ops.relpos_bias_1d(torch.zeros(32, 2), 4, 4), lambda: ops.relpos_bias_1d_backward(torch.zeros(1, 2, 4, 4), 32),
              lambda: ops.swin_relpos_bias_backward(torch.zeros(1, 2, 4, 4), 2)):
        with pytest.raises(_lib.OvisError, match="HIP device"):
            f()


@pytest.mark.parametrize("num,dist,both", [(32, 128, True), (32, 128, False), (8, 64, True), (64, 1000, True), (2, 2, False), (4, 2, True), (257, 100000, False)])
def test_bucket_borders(num, dist, both):
    """against the logarithm, away from where rounding could decide: bucket = e + floor(log(d / e) / log(dist / e) * (n - e))"""
    at = ops._relpos_borders(num, dist, both).tolist()
    cnt = len(at)
    n = num // 2 if both else num
    e = n // 2
    assert cnt == n - 1 and list(at) == sorted(at) and at[0] >= 1 and at[cnt - 1] <= dist
    for d in list(range(0, min(3 * dist, 5000))) + [10 ** 6]:
        mine = sum(d >= b for b in at)
        if d < e:
            assert mine == d
        else:
            v = e + math.log(d / e) / math.log(dist / e) * (n - e)
            if abs(v - round(v)) > 1e-9:
                assert mine == min(n - 1, int(v)), d
            else:                                    # a whole number by rights
                assert mine == min(n - 1, round(v)), d


def test_meta_tensors_give_shapes_and_types():
    m = lambda *s, t=torch.float16: torch.empty(*s, dtype=t, device="meta")
    g = m(96, t=torch.float32)
    o = ops.layernorm_forward(m(3, 5, 96), g, g, residual=m(3, 5, 96), checkpoint=True)
    assert o.y.shape == o.sum.shape == (3, 5, 96) and o.stats.shape == (15, 2) and o.xhat8.codes.shape == (15, 96) and o.xhat8.scales.shape == (15, 3)
    dx, dg, db = ops.layernorm_backward(m(3, 5, 96), o.xhat8, o.stats, g, out_dtype=torch.float32)
    assert dx.shape == (3, 5, 96) and dx.dtype == torch.float32 and dg.shape == db.shape == (96,)
    y, h8 = ops.act_forward_ckpt8(m(15, 40), ops.ACT_GELU)
    dh, dbias, y8 = ops.act_backward_ckpt8(m(15, 40), h8, ops.ACT_GELU, recompute=True)
    assert y.shape == dh.shape == (15, 40) and dbias.shape == (40,) and y8.scales.shape == (15, 2)
    dw, db = ops.linear_wgrad_ckpt8(m(15, 7), h8)
    assert dw.shape == (7, 40) and db.shape == (7,) and ops.ckpt8_decode(h8, torch.bfloat16).dtype == torch.bfloat16
    t = m(32, 4, t=torch.float32)
    assert ops.relpos_bias_1d(t, 3, 9, out_dtype=torch.float16).shape == (4, 3, 9) and ops.relpos_bias_1d(t, 3, 9, ld=12).shape == (4, 3, 12)
    assert ops.relpos_bias_1d_backward(m(2, 4, 3, 9), 32).shape == (32, 4) and ops.swin_relpos_bias_backward(m(2, 4, 9, 9), 3).shape == (25, 4)


@pytest.mark.parametrize("x", [lambda t: t(3, 1, 8).expand(3, 4, 8), lambda t: t(1, 4, 8).expand(3, 4, 8), lambda t: t(1, 8).expand(5, 8),
                               lambda t: t(5, 16)[:, ::2], lambda t: t(8, 5).t(), lambda t: t(4, 3, 8).transpose(0, 1), lambda t: t(3, 6, 8)[:, :4],
                               lambda t: t(5, 1).expand(5, 8), lambda t: t(1, 1).expand(5, 1), lambda t: t(40).as_strided((5, 8), (4, 1))])
def test_rows_that_are_not_one_stride_apart_are_refused(x):
    x = x(lambda *s: torch.empty(*s, device="meta"))
    g = torch.empty(x.shape[-1], device="meta")
    with pytest.raises(_lib.OvisError, match="one stride apart"):
        ops.layernorm_forward(x, g, g)
    with pytest.raises(_lib.OvisError, match="one stride apart"):
        ops.act_forward_ckpt8(x, ops.ACT_RELU)


@pytest.mark.parametrize("x", [lambda t: t(5, 24)[:, 8:16], lambda t: t(3, 4, 24)[..., :8], lambda t: t(9, 8)[::2], lambda t: t(3, 1, 24)[..., :8],
                               lambda t: t(1, 8).expand(1, 8), lambda t: t(5, 3)[:, 1:2], lambda t: t(0, 8), lambda t: t(8)])
def test_strided_rows_are_taken(x):
    x = x(lambda *s: torch.empty(*s, device="meta"))
    g = torch.empty(x.shape[-1], device="meta")
    assert ops.layernorm_forward(x, g, g).y.shape == x.shape


def test_no_autograd_graph_is_built():
    m = lambda *s: torch.empty(*s, device="meta", requires_grad=True)
    o = ops.layernorm_forward(m(5, 64), m(64), m(64), residual=m(5, 64), checkpoint=True)
    outs = [o.y, o.sum, o.stats, *ops.layernorm_backward(m(5, 64), o.xhat8, o.stats, m(64)), *ops.linear_wgrad_ckpt8(m(5, 7), o.xhat8),
            ops.act_forward_ckpt8(m(5, 64), ops.ACT_GELU)[0], ops.act_backward_ckpt8(m(5, 64), o.xhat8, ops.ACT_GELU)[0],
            ops.relpos_bias_1d(m(32, 4), 3, 9), ops.relpos_bias_1d_backward(m(4, 3, 9), 32), ops.swin_relpos_bias_backward(m(4, 9, 9), 3)]
    assert all(not t.requires_grad and t.grad_fn is None for t in outs)
