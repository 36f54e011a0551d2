"""What the training-side operators of `openvis_amd.ops` are measured on.

Four operators that a fine-tuning step of the framework's transformer blocks needs next to their forward passes:

  layer norm             `layernorm_forward` (with the row statistics, the sum with the residual, and the normalised rows in 8 bits) and
                         `layernorm_backward` (input, weight and bias gradients; from the rows or from their 8-bit form)
  relative position bias `relpos_bias_1d` (logarithmic buckets of the distance), `relpos_bias_1d_backward`, `swin_relpos_bias_backward`
  8-bit activations      `act_forward_ckpt8` / `act_backward_ckpt8`: the activation function of an MLP whose input is kept in 8 bits
  weight gradient        `linear_wgrad_ckpt8`: the gradient of a linear layer's weight and bias from its input in 8 bits

An 8-bit form is e4m3 codes with one power-of-two scale per 32 columns of a row.  With `own` false, `run` computes the operators by
elementary torch operations in 32 bits; with `own` true it calls the framework.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 32                                          # columns that share a scale
ACTS = {"relu": 1, "quickgelu": 2, "gelu": 3}       # the framework's activation codes


# ---- the cases ----------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # post-norm of a masked-attention decoder layer: 100 queries, f32, with its residual; one call of very little work
        dict(name="ln_fwd_queries", op="ln_fwd", rows=100, C=256, x="f32", y="f32", residual=True, ckpt=False),
        # pre-norm of the CLIP ViT-B/16 tower on 500 crops (197 tokens each), the fp16 residual stream, normalised rows kept in 8 bits
        dict(name="ln_fwd_tower", op="ln_fwd", rows=98500, C=768, x="f16", y="f16", residual=False, ckpt=True),
        # its backward pass from the 8-bit rows, the gradient of the residual stream added
        dict(name="ln_bwd_tower", op="ln_bwd", rows=98500, C=768, x="f16", y="f16", ckpt=True, dsum=True),
        # pre-norm of Swin-L's second stage on five 720p frames (92 x 160 tokens): f32 stream, fp16 branch, from the rows themselves
        dict(name="ln_bwd_swin", op="ln_bwd", rows=73600, C=384, x="f32", y="f16", ckpt=False, dsum=True),
        # the bias row of one new token against 4097 keys: a call that is all latency
        dict(name="relpos_fwd_token", op="relpos_fwd", H=16, Nq=1, Nk=4097, buckets=32, dist=128, both=False, off=4096, x="f32"),
        # the whole bias of a long sequence, both directions
        dict(name="relpos_fwd_long", op="relpos_fwd", H=16, Nq=4096, Nk=4096, buckets=32, dist=128, both=True, off=0, x="f16"),
        # Swin-L's first stage at 1080p: 920 windows of 12 x 12 tokens, 6 heads, gradient of the scores in f32
        dict(name="relpos_bwd_window", op="swin_bwd", B=920, H=6, ws=12, x="f32"),
        # a batch of eight odd-length causal sequences, bf16
        dict(name="relpos_bwd_odd", op="relpos_bwd", B=8, H=8, Nq=1023, Nk=1023, buckets=32, dist=128, both=False, off=0, x="bf16"),
        # fc1's output in the CLIP ViT-L/14@336 tower, 64 crops of 577 tokens
        dict(name="act_fwd_tower", op="act_fwd", rows=36928, C=4096, act="quickgelu", x="f16"),
        # the same place in Swin-L's second stage (GELU), backward, with the activation recomputed for fc2's weight gradient
        dict(name="act_bwd_swin", op="act_bwd", rows=73600, C=1536, act="gelu", x="f16", recompute=True),
        # fc2 of a decoder layer's FFN: 100 queries, f32
        dict(name="wgrad_queries", op="wgrad", M=100, N=256, K=2048, x="f32", fold=False),
        # fc2 of the ViT-L/14@336 tower, 64 crops
        dict(name="wgrad_tower", op="wgrad", M=36928, N=1024, K=4096, x="f16", fold=False),
    ]


def _spread(rng, lo, hi):
    """a whole number from lo to hi, spread over its logarithm"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "relpos_fwd", "relpos_bwd", "swin_bwd", "act_fwd", "act_bwd", "wgrad"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        t = rng.choice(["f32", "f16", "bf16"])
        if op in ("ln_fwd", "ln_bwd"):
            c = dict(op=op, rows=_spread(rng, 1, 100000), C=_spread(rng, 16, 4096), x=t, y=rng.choice(["f32", "f16", "bf16"]) if t == "f32" else t)
            c.update(dict(residual=rng.random() < 0.5, ckpt=rng.random() < 0.5) if op == "ln_fwd" else dict(ckpt=rng.random() < 0.5, dsum=rng.random() < 0.5))
        elif op in ("relpos_fwd", "relpos_bwd"):
            both = rng.random() < 0.5
            nk = _spread(rng, 1, 4096)
            nq = nk if rng.random() < 0.5 else _spread(rng, 1, 4096)
            buckets = rng.choice([8, 16, 32, 64])
            c = dict(op=op, H=_spread(rng, 1, 32), Nq=nq, Nk=nk, buckets=buckets, dist=rng.choice([64, 128, 256, 1000]), both=both,
                     off=max(0, nk - nq) if not both else 0, x=t)
            if op == "relpos_bwd":
                c["B"] = _spread(rng, 1, 16)
        elif op == "swin_bwd":
            c = dict(op=op, B=_spread(rng, 1, 4000), H=_spread(rng, 1, 48), ws=rng.randint(4, 16), x=t)
        elif op == "act_fwd":
            c = dict(op=op, rows=_spread(rng, 1, 100000), C=_spread(rng, 16, 8192), act=rng.choice(list(ACTS)), x=t)
        elif op == "act_bwd":
            c = dict(op=op, rows=_spread(rng, 1, 100000), C=_spread(rng, 16, 8192), act=rng.choice(list(ACTS)), x=t, recompute=rng.random() < 0.5)
        else:
            c = dict(op=op, M=_spread(rng, 1, 100000), N=_spread(rng, 8, 4096), K=_spread(rng, 16, 4096), x=t, fold=rng.random() < 0.3)
        if _cost(c) <= most:
            return c


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def work(case):
    op, x = case["op"], SIZE[case["x"]]
    if op in ("ln_fwd", "ln_bwd"):
        n, nb, y = case["rows"] * case["C"], case["rows"] * -(-case["C"] // BLOCK), SIZE[case["y"]]
        eight = n + nb
        if op == "ln_fwd":
            b = n * (x + y) + (2 * n * x if case["residual"] else 0) + (eight if case["ckpt"] else 0) + 8 * case["rows"] + 8 * case["C"]
            return {"bytes": b, "flops": 8.0 * n}
        b = n * (y + x) + (eight if case["ckpt"] else n * x) + (n * x if case["dsum"] else 0) + 8 * case["rows"] + 12 * case["C"]
        return {"bytes": b, "flops": 12.0 * n}
    if op == "relpos_fwd":
        n = case["H"] * case["Nq"] * case["Nk"]
        return {"bytes": n * x + 4 * case["H"] * case["buckets"], "flops": n}
    if op in ("relpos_bwd", "swin_bwd"):
        nq, nk = (case["ws"] ** 2,) * 2 if op == "swin_bwd" else (case["Nq"], case["Nk"])
        n = case["B"] * case["H"] * nq * nk
        return {"bytes": n * x + 4 * case["H"] * ((2 * case["ws"] - 1) ** 2 if op == "swin_bwd" else case["buckets"]), "flops": n}
    if op in ("act_fwd", "act_bwd"):
        n, nb = case["rows"] * case["C"], case["rows"] * -(-case["C"] // BLOCK)
        if op == "act_fwd":
            return {"bytes": 2 * n * x + n + nb, "flops": 10.0 * n}
        return {"bytes": 2 * n * x + (2 if case["recompute"] else 1) * (n + nb) + 4 * case["C"], "flops": 20.0 * n}
    M, N, K = case["M"], case["N"], case["K"]
    return {"bytes": M * N * x + M * K + M * -(-K // BLOCK) + 4 * N * K + 4 * N, "flops": 2.0 * M * N * K}


# ---- inputs -------------------------------------------------------------------------------------------------------------------------
def _stream(g, rows, C, dt):
    """rows of a residual stream: unit noise around a mean of each channel's own, a few channels much larger than the others"""
    size = torch.exp(0.5 * torch.randn(C, generator=g, device="cuda"))
    size[torch.randint(0, C, (max(1, C // 100),), generator=g, device="cuda")] *= 12.0
    v = torch.randn(rows, C, generator=g, device="cuda")
    return v.mul_(size).add_(0.3 * torch.randn(C, generator=g, device="cuda")).to(dt)


def _grad(g, shape, dt):
    """a loss-scaled gradient"""
    return torch.randn(shape, generator=g, device="cuda").mul_(0.25).to(dt)


def _quantise(v, signed_zero=False):
    """f32 rows -> (e4m3 codes, e8m0 scales [rows, ceil(C / 32)]): the smallest power of two under which the block's largest finite value is
    at most 448.  signed_zero: the sign of a code says whether the value was positive (ReLU's derivative)."""
    R, C = v.shape
    nb = -(-C // BLOCK)
    p = torch.nn.functional.pad(v, (0, nb * BLOCK - C)).view(R, nb, BLOCK)
    a = p.abs()
    a = torch.where(torch.isfinite(a), a, torch.zeros_like(a)).amax(-1)
    m, e = torch.frexp(a)
    sh = torch.where(a > 0, e - 9 + (m > 0.875).int(), torch.full_like(e, -100)).clamp(-100, 120)
    q = p * ((127 - sh) << 23).view(torch.float32)[..., None]
    q = torch.where(torch.isinf(q), torch.full_like(q, math.nan), q)
    if signed_zero:
        q = torch.where(p == 0, torch.full_like(q, -0.0), q)
    codes = q.to(torch.float8_e4m3fn).view(R, nb * BLOCK)[:, :C].contiguous()
    return codes, (sh + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _value(codes, scales):
    """the f32 values that an 8-bit form stands for"""
    C = codes.shape[1]
    return codes.float() * scales.float().repeat_interleave(BLOCK, dim=1)[:, :C]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, s = case["op"], dict(case=case)
    dt = DT[case["x"]]
    if op in ("ln_fwd", "ln_bwd"):
        R, C = case["rows"], case["C"]
        s["gamma"] = 1.0 + 0.2 * torch.randn(C, generator=g, device="cuda")
        s["beta"] = 0.2 * torch.randn(C, generator=g, device="cuda")
        x = _stream(g, R, C, dt)
        if op == "ln_fwd":
            s["x"] = x
            s["residual"] = _stream(g, R, C, dt) if case["residual"] else None
            return s
        f = x.float()
        mean = f.mean(1, keepdim=True)
        rstd = torch.rsqrt(((f - mean) ** 2).mean(1, keepdim=True) + 1e-5)
        s["stats"] = torch.cat((mean, rstd), 1).contiguous()
        s["x"] = _quantise((f - mean) * rstd) if case["ckpt"] else x
        s["dy"] = _grad(g, (R, C), DT[case["y"]])
        s["dsum"] = _grad(g, (R, C), dt) if case["dsum"] else None
    elif op == "relpos_fwd":
        s["table"] = torch.randn(case["buckets"], case["H"], generator=g, device="cuda")
    elif op == "relpos_bwd":
        s["dbias"] = _grad(g, (case["B"], case["H"], case["Nq"], case["Nk"]), dt)
        if not case["both"]:                        # behind the query nothing was attended to
            i = torch.arange(case["Nq"], device="cuda")[:, None] + case["off"]
            s["dbias"] *= torch.arange(case["Nk"], device="cuda")[None, :] <= i
    elif op == "swin_bwd":
        s["dbias"] = _grad(g, (case["B"], case["H"], case["ws"] ** 2, case["ws"] ** 2), dt)
    elif op == "act_fwd":
        s["h"] = torch.randn(case["rows"], case["C"], generator=g, device="cuda").mul_(1.5).sub_(0.3).to(dt)
    elif op == "act_bwd":
        h = torch.randn(case["rows"], case["C"], generator=g, device="cuda").mul_(1.5).sub_(0.3).to(dt)
        s["h8"] = _quantise(h.float(), case["act"] == "relu")
        s["dy"] = _grad(g, h.shape, dt)
    else:
        s["x8"] = _quantise(_stream(g, case["M"], case["K"], torch.float32))
        s["dy"] = _grad(g, (case["M"], case["N"]), dt)
        s["gamma"] = 1.0 + 0.2 * torch.randn(case["K"], generator=g, device="cuda") if case["fold"] else None
        s["beta"] = 0.2 * torch.randn(case["K"], generator=g, device="cuda") if case["fold"] else None
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    return (_own if own else _plain)(c["op"], c, s)


def _own(op, c, s):
    from openvis_amd import ops
    if op == "ln_fwd":
        r = ops.layernorm_forward(s["x"], s["gamma"], s["beta"], residual=s["residual"], out_dtype=DT[c["y"]], checkpoint=c["ckpt"])
        return {"y": r.y, "sum": r.sum if c["residual"] else None, "stats": r.stats,
                "codes": r.xhat8.codes if c["ckpt"] else None, "scales": r.xhat8.scales if c["ckpt"] else None}
    if op == "ln_bwd":
        x = ops.Ckpt8(*s["x"]) if c["ckpt"] else s["x"]
        dx, dgamma, dbeta = ops.layernorm_backward(s["dy"], x, s["stats"], s["gamma"], dsum=s["dsum"], out_dtype=DT[c["x"]])
        return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if op == "relpos_fwd":
        return ops.relpos_bias_1d(s["table"], c["Nq"], c["Nk"], max_distance=c["dist"], bidirectional=c["both"], q_offset=c["off"],
                                  out_dtype=DT[c["x"]])
    if op == "relpos_bwd":
        return ops.relpos_bias_1d_backward(s["dbias"], c["buckets"], max_distance=c["dist"], bidirectional=c["both"], q_offset=c["off"])
    if op == "swin_bwd":
        return ops.swin_relpos_bias_backward(s["dbias"], c["ws"])
    if op == "act_fwd":
        y, h8 = ops.act_forward_ckpt8(s["h"], ACTS[c["act"]])
        return {"y": y, "codes": h8.codes, "scales": h8.scales}
    if op == "act_bwd":
        dh, dbias, y8 = ops.act_backward_ckpt8(s["dy"], ops.Ckpt8(*s["h8"]), ACTS[c["act"]], recompute=c["recompute"])
        return {"dh": dh, "dbias": dbias, "codes": y8.codes if c["recompute"] else None, "scales": y8.scales if c["recompute"] else None}
    dw, db = ops.linear_wgrad_ckpt8(s["dy"], ops.Ckpt8(*s["x8"]), gamma=s["gamma"], beta=s["beta"])
    return {"dw": dw, "db": db}


def _bucket_1d(r, c, like):
    """bucket of the distance r = key position - query position: one bucket a step up to half the buckets of a direction, then
    logarithmically wider ones up to the distance `dist`, the last for all that is farther.  The borders are counted in 64 bits; those that
    are whole numbers by rights (a root of a whole number) get a hair's breadth, so that rounding does not push them down."""
    nb = c["buckets"] // 2 if c["both"] else c["buckets"]
    n = r.abs() if c["both"] else (-r).clamp(min=0)
    exact_n = nb // 2
    far = exact_n + torch.floor(torch.log(n.clamp(min=1).double() / exact_n) / math.log(c["dist"] / exact_n) * (nb - exact_n) + 1e-9).long()
    b = torch.where(n < exact_n, n, far.clamp(max=nb - 1))
    return b + nb * (r > 0).long() if c["both"] else b


def _diagonals(d):
    """[..., n, m] -> [..., n + m - 1]: the sums over the diagonals, of column - row + n - 1.  Rows last to first, padded to n + m and read
    again as rows one shorter, so that a diagonal becomes a column"""
    n, m = d.shape[-2:]
    w = n + m
    d = torch.nn.functional.pad(d.flip(-2), (0, n)).flatten(-2)[..., :n * (w - 1)]
    return d.unflatten(-1, (n, w - 1)).sum(-2)


def _act(h, name):
    if name == "relu":
        return h.clamp(min=0)
    if name == "quickgelu":
        return h * torch.sigmoid(1.702 * h)
    return 0.5 * h * (1.0 + torch.erf(h * math.sqrt(0.5)))


def _act_slope(h, name):
    """the derivative at the value that an 8-bit form stands for"""
    if name == "relu":
        return (~torch.signbit(h)).to(h.dtype)
    if name == "quickgelu":
        g = torch.sigmoid(1.702 * h)
        return g * (1.0 + 1.702 * h * (1.0 - g))
    return 0.5 * (1.0 + torch.erf(h * math.sqrt(0.5))) + h * torch.exp(-0.5 * h * h) * (1.0 / math.sqrt(2 * math.pi))


def _plain(op, c, s):
    dt = DT[c["x"]]
    if op == "ln_fwd":
        x = s["x"]
        total = (x.float() + s["residual"].float()).to(dt) if c["residual"] else None
        f = (total if c["residual"] else x).float()
        mean = f.mean(1, keepdim=True)
        d = f - mean
        rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5)
        xhat = d * rstd
        codes, scales = _quantise(xhat) if c["ckpt"] else (None, None)
        return {"y": (xhat * s["gamma"] + s["beta"]).to(DT[c["y"]]), "sum": total, "stats": torch.cat((mean, rstd), 1), "codes": codes, "scales": scales}
    if op == "ln_bwd":
        dy, mean, rstd = s["dy"].float(), s["stats"][:, :1], s["stats"][:, 1:]
        xhat = _value(*s["x"]) if c["ckpt"] else (s["x"].float() - mean) * rstd
        gd = dy * s["gamma"]
        dx = rstd * (gd - gd.mean(1, keepdim=True) - xhat * (gd * xhat).mean(1, keepdim=True))
        if c["dsum"]:
            dx = dx + s["dsum"].float()
        return {"dx": dx.to(dt), "dgamma": (dy * xhat).sum(0), "dbeta": dy.sum(0)}
    if op == "relpos_fwd":
        r = torch.arange(c["Nk"], device="cuda")[None, :] - torch.arange(c["Nq"], device="cuda")[:, None] - c["off"]
        return s["table"].t().to(dt)[:, _bucket_1d(r, c, s["table"])]
    if op == "relpos_bwd":
        Nq, Nk = c["Nq"], c["Nk"]
        d = _diagonals(s["dbias"].sum(0, dtype=torch.float32))
        b = _bucket_1d(torch.arange(Nq + Nk - 1, device="cuda") - (Nq - 1) - c["off"], c, d)
        return torch.matmul(torch.nn.functional.one_hot(b, c["buckets"]).t().double(), d.t().double()).float()
    if op == "swin_bwd":
        ws, H = c["ws"], c["H"]
        d = s["dbias"].sum(0, dtype=torch.float32).view(H, ws, ws, ws, ws)                   # [H, yi, xi, yj, xj]
        d = _diagonals(d.permute(0, 2, 4, 3, 1).contiguous())                                # [H, xi, xj, yi - yj + ws - 1]
        d = _diagonals(d.permute(0, 3, 2, 1).contiguous())                                   # [H, yi - yj + ws - 1, xi - xj + ws - 1]
        return d.reshape(H, -1).t().contiguous()
    if op == "act_fwd":
        h = s["h"].float()
        codes, scales = _quantise(h, c["act"] == "relu")
        return {"y": _act(h, c["act"]).to(dt), "codes": codes, "scales": scales}
    if op == "act_bwd":
        h = _value(*s["h8"])
        dh = s["dy"].float() * _act_slope(h, c["act"])
        codes, scales = _quantise(_act(h, c["act"])) if c["recompute"] else (None, None)
        return {"dh": dh.to(dt), "dbias": dh.sum(0), "codes": codes, "scales": scales}
    dy = s["dy"].float()
    dw, db = torch.matmul(dy.t(), _value(*s["x8"])), dy.sum(0)
    if c["fold"]:
        dw = dw * s["gamma"] + db[:, None] * s["beta"]
    return {"dw": dw, "db": db}


# ---- the same from the definitions, in 64 bits --------------------------------------------------------------------------------------
def _pow2(k):
    return ((k.long() + 1023) << 52).view(torch.float64)


def _quantise64(v):
    R, C = v.shape
    nb = -(-C // BLOCK)
    u = torch.zeros(R, nb * BLOCK, dtype=torch.float64, device=v.device)
    u[:, :C] = v
    u = u.view(R, nb, BLOCK)
    top = u.abs().max(-1, keepdim=True).values.clamp(min=1e-300)
    k = torch.ceil(torch.log2(top / 448.0)).long()
    k = k + (top > 448.0 * _pow2(k)).long() - (top <= 448.0 * _pow2(k - 1)).long()
    k = k.clamp(-100, 120)
    u = u / _pow2(k)
    step = _pow2((torch.frexp(u)[1] - 1).clamp(min=-6) - 3)
    return (torch.round(u / step) * step).view(R, nb * BLOCK)[:, :C].contiguous(), _pow2(k).squeeze(-1)


def _value64(codes, scales):
    s = scales.double()[:, :, None].expand(-1, -1, BLOCK).reshape(codes.shape[0], -1)
    return codes.double() * s[:, :codes.shape[1]]


def _gauss_cdf64(h):
    return 0.5 * torch.erfc(-h / math.sqrt(2.0))


def exact(case, seed):
    c, s = case, prepare(case, seed)
    op, dt = c["op"], DT[c["x"]]
    if op == "ln_fwd":
        x = s["x"].double()
        total = (x + s["residual"].double()).float().to(dt) if c["residual"] else None
        v = (total if c["residual"] else s["x"]).double()
        mean = v.sum(1) / c["C"]
        var = (v - mean[:, None]).pow(2).sum(1) / c["C"]
        rstd = (var + 1e-5).pow(-0.5)
        xhat = (v - mean[:, None]) * rstd[:, None]
        codes, scales = _quantise64(xhat) if c["ckpt"] else (None, None)
        return {"y": xhat * s["gamma"].double() + s["beta"].double(), "sum": None if total is None else total.double(),
                "stats": torch.stack((mean, rstd), 1), "codes": codes, "scales": scales}
    if op == "ln_bwd":
        dy, mean, rstd = s["dy"].double(), s["stats"][:, 0].double()[:, None], s["stats"][:, 1].double()[:, None]
        xhat = _value64(*s["x"]) if c["ckpt"] else (s["x"].double() - mean) * rstd
        gd = dy * s["gamma"].double()
        dx = rstd * (gd - gd.sum(1, keepdim=True) / c["C"] - xhat * ((gd * xhat).sum(1, keepdim=True) / c["C"]))
        return {"dx": dx + (s["dsum"].double() if c["dsum"] else 0.0), "dgamma": torch.einsum("rc,rc->c", dy, xhat), "dbeta": dy.sum(0)}
    if op in ("relpos_fwd", "relpos_bwd"):
        H, Nq, Nk = c["H"], c["Nq"], c["Nk"]
        side = c["buckets"] // 2 if c["both"] else c["buckets"]
        half = side // 2
        # the first distance of each bucket of a direction, from whole numbers alone: n belongs to half + k or beyond when
        # (n / half) ** (side - half) >= (dist / half) ** k
        first = list(range(half)) + [half]
        for k in range(1, side - half):
            n = first[-1]
            while n ** (side - half) * half ** k < c["dist"] ** k * half ** (side - half):
                n += 1
            first.append(n)
        of = torch.zeros(Nq + Nk + abs(c["off"]) + 1, dtype=torch.long)
        for b, n in enumerate(first):
            of[n:] = b
        r = torch.arange(-(Nq - 1), Nk) - c["off"]
        bucket = (of[r.abs()] + side * (r > 0) if c["both"] else of[(-r).clamp(min=0)]).cuda()      # of the diagonals, key - query ascending
        if op == "relpos_fwd":
            line = s["table"].double().t().contiguous()[:, bucket]                                   # [H, diagonals]
            return line.unfold(1, Nk, 1).flip(1)                                                     # row i starts at diagonal Nq - 1 - i
        out = torch.zeros(c["buckets"], H, dtype=torch.float64, device="cuda")
        for i in range(Nq):
            out.index_add_(0, bucket[Nq - 1 - i:Nq - 1 - i + Nk], s["dbias"][:, :, i].sum(0, dtype=torch.float64).t())
        return out
    if op == "swin_bwd":
        ws, H = c["ws"], c["H"]
        d = s["dbias"].sum(0, dtype=torch.float64).view(H, ws, ws, ws, ws)                           # [H, yi, xi, yj, xj]
        out = torch.zeros(2 * ws - 1, 2 * ws - 1, H, dtype=torch.float64, device="cuda")
        for yi in range(ws):
            for xi in range(ws):
                out[yi:yi + ws, xi:xi + ws] += d[:, yi, xi].flip(1, 2).permute(1, 2, 0)              # yi - yj + ws - 1 falls from yi + ws - 1 to yi
        return out.view(-1, H)
    if op == "act_fwd":
        h = s["h"].double()
        y = torch.relu(h) if c["act"] == "relu" else h / (1.0 + torch.exp(-1.702 * h)) if c["act"] == "quickgelu" else h * _gauss_cdf64(h)
        codes, scales = _quantise64(h)
        return {"y": y, "codes": codes, "scales": scales}
    if op == "act_bwd":
        h = _value64(*s["h8"])
        if c["act"] == "relu":
            y, slope = torch.relu(h), torch.where(torch.signbit(h), 0.0, 1.0).double()
        elif c["act"] == "quickgelu":
            e = 1.0 / (1.0 + torch.exp(-1.702 * h))
            y, slope = h * e, e + 1.702 * h * e * (1.0 - e)
        else:
            y = h * _gauss_cdf64(h)
            slope = _gauss_cdf64(h) + h * torch.exp(-h * h / 2) / math.sqrt(2 * math.pi)
        dh = s["dy"].double() * slope
        codes, scales = _quantise64(y) if c["recompute"] else (None, None)
        return {"dh": dh, "dbias": dh.sum(0), "codes": codes, "scales": scales}
    dy, x = s["dy"].double(), _value64(*s["x8"])
    dw, db = dy.t().contiguous() @ x, dy.sum(0)
    if c["fold"]:
        dw = dw * s["gamma"].double()[None, :] + db[:, None] * s["beta"].double()[None, :]
    return {"dw": dw, "db": db}
