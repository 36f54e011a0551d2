// Dispatcher ops `ovis_mi::*` of the training-side operators (layer norm, relative position bias, 8-bit activations, weight gradient): checks of
// the arguments, outputs and workspaces from torch's allocator, one C entry point each on the device's CURRENT stream.  openvis_amd/ops.py
// calls these; from Python alone a small call costs 9 to 14 us on the host, half of it allocations and conversions, from here 6 to 10.
// The same functions serve meta tensors (shapes and types only).  No arithmetic here.
#include <torch/extension.h>
#include <torch/library.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include "../../../include/openvis_hip.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;
using OptType = c10::optional<at::ScalarType>;

ovis_stream_t cur_stream() { return (ovis_stream_t)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }
const Tensor* opt(const OptTensor& t) { return t.has_value() && t->defined() ? &*t : nullptr; }

// every tensor on one HIP (or meta) device; the guard makes it the current one, so that its current stream is used
struct On {
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard;
  bool meta;
  On(const char* name, std::initializer_list<const Tensor*> ts) : meta(false) {
    const Tensor* first = nullptr;
    for (const Tensor* t : ts) {
      if (!t) continue;
      TORCH_CHECK(t->is_cuda() || t->is_meta(), name, ": tensors must be on a HIP device (got ", t->device(), "; no CPU fallback)");
      if (!first) first = t;
      TORCH_CHECK(t->device() == first->device(), name, ": tensors must be on one HIP device (got ", first->device(), " and ", t->device(), ")");
    }
    meta = first->is_meta();
    if (!meta) guard.reset_device(first->device());
  }
};

void done(const char* name, int rc) { TORCH_CHECK(rc == OVIS_OK, name, ": ", ovis_last_error()); }

int code(const char* name, const char* what, at::ScalarType t) {
  TORCH_CHECK(t == at::kFloat || t == at::kHalf || t == at::kBFloat16, name, ": ", what, " must be float32, float16 or bfloat16");
  return t == at::kFloat ? OVIS_F32 : t == at::kHalf ? OVIS_F16 : OVIS_BF16;
}

struct Rows { int64_t n, ld; };
// t [..., C] as rows that are one stride apart, elements contiguous
Rows rows_of(const char* name, const char* what, const Tensor& t, int64_t C) {
  TORCH_CHECK(t.dim() >= 1 && C >= 1 && t.size(-1) == C, name, ": ", what, " must be [..., ", C, "], got ", t.sizes());
  const int64_t n = t.numel() / C;
  if (t.is_contiguous()) return {n, C};
  bool ok = C == 1 || t.stride(-1) == 1;
  int64_t ld = C, next = -1;                                     // stride of the innermost leading dimension, and what the next one's must be
  for (int64_t d = t.dim() - 2; d >= 0 && ok; --d) {
    if (t.size(d) == 1) continue;
    if (next < 0) ld = t.stride(d);                              // 0 for an expanded dimension: refused below
    else ok = t.stride(d) == next;
    next = t.stride(d) * t.size(d);
  }
  TORCH_CHECK(ok && ld >= C, name, ": ", what, " needs contiguous elements in rows that are one stride apart (got strides ", t.strides(), ")");
  return {n, ld};
}

void vec(const char* name, const char* what, const Tensor& t, int64_t C) {
  TORCH_CHECK(t.scalar_type() == at::kFloat && t.numel() == C && t.is_contiguous(), name, ": ", what, " must be a contiguous float32 vector of ", C);
}
const float* f32(const Tensor* t) { return t ? t->const_data_ptr<float>() : nullptr; }
const void* ptr(const Tensor* t) { return t ? t->const_data_ptr() : nullptr; }
Tensor floats(const Tensor& like, at::IntArrayRef s) { return at::empty(s, like.options().dtype(at::kFloat)); }
Tensor words(const Tensor& like, long long bytes) { return at::empty({(int64_t)(bytes / 4)}, like.options().dtype(at::kFloat)); }
Tensor same(const Tensor& t, at::ScalarType type) { return at::empty(t.sizes(), t.options().dtype(type)); }

// the two tensors of the 8-bit form
struct Eight {
  Tensor codes, scales;
  static Eight make(const Tensor& like, int64_t rows, int64_t C) {
    return {at::empty({rows, C}, like.options().dtype(at::kFloat8_e4m3fn)), at::empty({rows, (C + 31) / 32}, like.options().dtype(at::kFloat8_e8m0fnu))};
  }
};
uint8_t* bytes(Tensor& t) { return t.defined() ? (uint8_t*)t.data_ptr() : nullptr; }
const uint8_t* cbytes(const Tensor* t) { return t ? (const uint8_t*)t->const_data_ptr() : nullptr; }
void check8(const char* name, const Tensor& codes, const Tensor& scales) {
  TORCH_CHECK(codes.scalar_type() == at::kFloat8_e4m3fn && scales.scalar_type() == at::kFloat8_e8m0fnu && codes.dim() == 2 && codes.is_contiguous() &&
                  scales.is_contiguous() && codes.size(1) >= 1 && scales.dim() == 2 && scales.size(0) == codes.size(0) &&
                  scales.size(1) == (codes.size(1) + 31) / 32,
              name, ": a Ckpt8 holds contiguous float8_e4m3fn codes [rows, C] and float8_e8m0fnu scales [rows, ceil(C / 32)]");
}
int small(const char* name, int64_t v) {
  TORCH_CHECK(v >= 0 && v < (1ll << 31), name, ": a size of ", v);
  return (int)v;
}

// -> y, sum (undefined without a residual), stats, codes, scales (undefined without checkpoint)
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> layernorm_forward(const Tensor& x, const Tensor& gamma, const Tensor& beta, const OptTensor& residual,
                                                                     double eps, OptType out_dtype, bool checkpoint) {
  const char* name = "layernorm_forward";
  const Tensor* res = opt(residual);
  On on(name, {&x, &gamma, &beta, res});
  const int xd = code(name, "x", x.scalar_type());
  const at::ScalarType yt = out_dtype.value_or(x.scalar_type());
  const int yd = code(name, "out_dtype", yt);
  const int64_t C = x.dim() ? x.size(-1) : 0;
  const Rows rx = rows_of(name, "x", x, C);
  Rows rr{0, 0};
  if (res) {
    TORCH_CHECK(res->scalar_type() == x.scalar_type() && res->sizes() == x.sizes(), name, ": residual must have x's shape and type");
    rr = rows_of(name, "residual", *res, C);
  }
  vec(name, "gamma", gamma, C);
  vec(name, "beta", beta, C);
  TORCH_CHECK(xd == OVIS_F32 || xd == yd, name, ": y has x's type, or any where x is float32");
  Tensor y = same(x, yt), sum = res ? same(x, x.scalar_type()) : Tensor(), stats = floats(x, {rx.n, 2});
  Eight e;
  if (checkpoint) e = Eight::make(x, rx.n, C);
  if (!on.meta && rx.n)
    done(name, ovis_layernorm_train_forward(x.const_data_ptr(), rx.ld, ptr(res), rr.ld, f32(&gamma), f32(&beta), res ? sum.data_ptr() : nullptr, y.data_ptr(),
                                            stats.data_ptr<float>(), bytes(e.codes), bytes(e.scales), rx.n, small(name, C), (float)eps, xd, yd, cur_stream()));
  return {y, sum, stats, e.codes, e.scales};
}

// x, or codes and scales -> dx, dgamma, dbeta
std::tuple<Tensor, Tensor, Tensor> layernorm_backward(const Tensor& dy, const OptTensor& x, const OptTensor& codes, const OptTensor& scales,
                                                      const Tensor& stats, const Tensor& gamma, const OptTensor& dsum, OptType out_dtype) {
  const char* name = "layernorm_backward";
  const Tensor *tx = opt(x), *tc = opt(codes), *ts = opt(scales), *ds = opt(dsum);
  TORCH_CHECK(!tx != !tc && !tc == !ts, name, ": the rows, or their 8-bit form");
  On on(name, {&dy, tx, tc, ts, &stats, &gamma, ds});
  const int dyd = code(name, "dy", dy.scalar_type());
  const int64_t C = dy.dim() ? dy.size(-1) : 0;
  const Rows rd = rows_of(name, "dy", dy, C);
  Rows rx{0, 0}, rs{0, 0};
  at::ScalarType xt;
  if (tc) {
    check8(name, *tc, *ts);
    TORCH_CHECK(tc->size(0) == rd.n && tc->size(1) == C, name, ": the 8-bit rows are ", tc->sizes(), ", dy has ", rd.n, " rows of ", C);
    xt = out_dtype.value_or(ds ? ds->scalar_type() : dy.scalar_type());
  } else {
    rx = rows_of(name, "x", *tx, C);
    TORCH_CHECK(rx.n == rd.n, name, ": x has ", rx.n, " rows, dy ", rd.n);
    xt = tx->scalar_type();
    TORCH_CHECK(out_dtype.value_or(xt) == xt, name, ": dx has x's type");
  }
  const int xd = code(name, "x / dx", xt);
  TORCH_CHECK(xd == OVIS_F32 || xd == dyd, name, ": dy has dx's type, or any where dx is float32");
  if (ds) {
    rs = rows_of(name, "dsum", *ds, C);
    TORCH_CHECK(ds->scalar_type() == xt && rs.n == rd.n, name, ": dsum must have dx's type and rows");
  }
  TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.numel() == 2 * rd.n && stats.is_contiguous(), name, ": stats must be contiguous float32 [", rd.n, ", 2]");
  vec(name, "gamma", gamma, C);
  Tensor dx = same(dy, xt), grads = rd.n ? floats(dy, {2, C}) : at::zeros({2, C}, dy.options().dtype(at::kFloat));
  Tensor dgamma = grads.select(0, 0), dbeta = grads.select(0, 1);
  if (!on.meta && rd.n) {
    const int c = small(name, C);
    Tensor ws = words(dy, ovis_layernorm_train_backward_workspace_bytes(rd.n, c, xd));
    float* g = grads.data_ptr<float>();
    done(name, ovis_layernorm_train_backward(dy.const_data_ptr(), rd.ld, ptr(tx), rx.ld, cbytes(tc), cbytes(ts), f32(&stats), f32(&gamma), ptr(ds), rs.ld,
                                             dx.data_ptr(), g, g + C, ws.data_ptr<float>(), rd.n, c, dyd, xd, cur_stream()));
  }
  return {dx, dgamma, dbeta};
}

// act 0: the 8-bit form alone, y undefined
std::tuple<Tensor, Tensor, Tensor> act_forward_ckpt8(const Tensor& h, int64_t act) {
  const char* name = act ? "act_forward_ckpt8" : "ckpt8_encode";
  On on(name, {&h});
  TORCH_CHECK(act >= 0 && act <= 3, name, ": act must be ACT_RELU, ACT_QUICKGELU or ACT_GELU");
  const int d = code(name, "input", h.scalar_type());
  const int64_t C = h.dim() ? h.size(-1) : 0;
  const Rows r = rows_of(name, "input", h, C);
  Tensor y = act ? same(h, h.scalar_type()) : Tensor();
  Eight e = Eight::make(h, r.n, C);
  if (!on.meta && r.n)
    done(name, ovis_act_ckpt8_forward(h.const_data_ptr(), r.ld, act ? y.data_ptr() : nullptr, bytes(e.codes), bytes(e.scales), r.n, small(name, C), (int)act, d,
                                      cur_stream()));
  return {y, e.codes, e.scales};
}

// -> dh, dbias, codes, scales of the activation (undefined without recompute)
std::tuple<Tensor, Tensor, Tensor, Tensor> act_backward_ckpt8(const Tensor& dy, const Tensor& codes, const Tensor& scales, int64_t act, bool recompute) {
  const char* name = "act_backward_ckpt8";
  On on(name, {&dy, &codes, &scales});
  TORCH_CHECK(act >= 1 && act <= 3, name, ": act must be ACT_RELU, ACT_QUICKGELU or ACT_GELU");
  check8(name, codes, scales);
  const int64_t rows = codes.size(0), C = codes.size(1);
  const int d = code(name, "dy", dy.scalar_type());
  const Rows r = rows_of(name, "dy", dy, C);
  TORCH_CHECK(r.n == rows, name, ": dy has ", r.n, " rows, the 8-bit rows are ", rows);
  Tensor dh = same(dy, dy.scalar_type()), db = rows ? floats(dy, {C}) : at::zeros({C}, dy.options().dtype(at::kFloat));
  Eight e;
  if (recompute) e = Eight::make(dy, rows, C);
  if (!on.meta && rows) {
    const int c = small(name, C);
    Tensor ws = words(dy, ovis_act_ckpt8_backward_workspace_bytes(rows, c));
    done(name, ovis_act_ckpt8_backward(dy.const_data_ptr(), r.ld, cbytes(&codes), cbytes(&scales), dh.data_ptr(), db.data_ptr<float>(), bytes(e.codes),
                                       bytes(e.scales), ws.data_ptr<float>(), rows, c, (int)act, d, cur_stream()));
  }
  return {dh, db, e.codes, e.scales};
}

Tensor ckpt8_decode(const Tensor& codes, const Tensor& scales, at::ScalarType dtype) {
  const char* name = "ckpt8_decode";
  On on(name, {&codes, &scales});
  check8(name, codes, scales);
  const int d = code(name, "dtype", dtype);
  Tensor out = same(codes, dtype);
  if (!on.meta && codes.size(0))
    done(name, ovis_ckpt8_decode(cbytes(&codes), cbytes(&scales), out.data_ptr(), codes.size(0), small(name, codes.size(1)), d, cur_stream()));
  return out;
}

std::tuple<Tensor, Tensor> linear_wgrad_ckpt8(const Tensor& dy, const Tensor& codes, const Tensor& scales, const OptTensor& gamma, const OptTensor& beta) {
  const char* name = "linear_wgrad_ckpt8";
  const Tensor *g = opt(gamma), *b = opt(beta);
  On on(name, {&dy, &codes, &scales, g, b});
  check8(name, codes, scales);
  const int64_t rows = codes.size(0), K = codes.size(1), N = dy.dim() ? dy.size(-1) : 0;
  const int d = code(name, "dy", dy.scalar_type());
  const Rows r = rows_of(name, "dy", dy, N);
  TORCH_CHECK(r.n == rows, name, ": dy has ", r.n, " rows, the 8-bit rows are ", rows);
  TORCH_CHECK(!g == !b, name, ": gamma and beta go together");
  if (g) {
    vec(name, "gamma", *g, K);
    vec(name, "beta", *b, K);
  }
  const auto o = dy.options().dtype(at::kFloat);
  if (!rows) return {at::zeros({N, K}, o), at::zeros({N}, o)};
  Tensor dw = at::empty({N, K}, o), db = at::empty({N}, o);
  if (!on.meta) {
    const int n = small(name, N), k = small(name, K);
    Tensor ws = words(dy, ovis_linear_wgrad_ckpt8_workspace_bytes(rows, n, k, d));
    done(name, ovis_linear_wgrad_ckpt8(dy.const_data_ptr(), r.ld, cbytes(&codes), cbytes(&scales), f32(g), f32(b), dw.data_ptr<float>(), db.data_ptr<float>(),
                                       ws.data_ptr<float>(), rows, n, k, d, cur_stream()));
  }
  return {dw, db};
}

// borders: int32 on the host (see the C entry point); ld: 0 = rows padded to 16 bytes and a view of the columns, else the padded rows themselves
Tensor relpos_bias_1d(const Tensor& table, const Tensor& borders, bool both, int64_t Nq, int64_t Nk, int64_t q_offset, at::ScalarType dtype, int64_t ld) {
  const char* name = "relpos_bias_1d";
  On on(name, {&table});
  const int nb = small(name, borders.numel());
  TORCH_CHECK(borders.device().is_cpu() && borders.scalar_type() == at::kInt && borders.is_contiguous(), name, ": borders int32 on the host");
  TORCH_CHECK(table.dim() == 2 && table.scalar_type() == at::kFloat && table.is_contiguous() && table.size(1) >= 1 && table.size(0) == (nb + 1) * (both ? 2 : 1),
              name, ": table must be contiguous float32 [buckets, heads]");
  const int d = code(name, "out_dtype", dtype);
  TORCH_CHECK(Nq >= 0 && Nk >= 0, name, ": Nq ", Nq, ", Nk ", Nk);
  const int64_t H = table.size(1), v = d == OVIS_F32 ? 4 : 8, row = ld ? ld : (Nk + v - 1) / v * v;
  TORCH_CHECK(row >= Nk && row % v == 0, name, ": ld must be at least ", Nk, " and a multiple of ", v);
  Tensor out = at::empty({H, Nq, row}, table.options().dtype(dtype));
  if (!on.meta) {
    if (Nq && Nk)
      done(name, ovis_relpos_bias_1d(f32(&table), out.data_ptr(), borders.const_data_ptr<int>(), nb, both, small(name, H), small(name, Nq), small(name, Nk),
                                     small(name, row), q_offset, d, cur_stream()));
    else if (out.numel())
      out.zero_();
  }
  return ld || row == Nk ? out : out.narrow(2, 0, Nk);
}

struct Grad { int64_t B, H, Nq, Nk, bs, hs, ld; };
Grad grad_of(const char* name, const Tensor& t) {
  TORCH_CHECK(t.dim() == 3 || t.dim() == 4, name, ": dbias must be [H, Nq, Nk] or [B, H, Nq, Nk], got ", t.sizes());
  const bool b = t.dim() == 4;
  Grad g{b ? t.size(0) : 1, t.size(-3), t.size(-2), t.size(-1), b ? t.stride(0) : 0, t.stride(-3), t.stride(-2)};
  TORCH_CHECK(g.H >= 1 && (g.Nk <= 1 || t.stride(-1) == 1), name, ": dbias needs contiguous rows (got ", t.sizes(), ", strides ", t.strides(), ")");
  return g;
}

Tensor relpos_bias_1d_backward(const Tensor& dbias, const Tensor& borders, bool both, int64_t q_offset) {
  const char* name = "relpos_bias_1d_backward";
  On on(name, {&dbias});
  const int d = code(name, "dbias", dbias.scalar_type()), nb = small(name, borders.numel());
  TORCH_CHECK(borders.device().is_cpu() && borders.scalar_type() == at::kInt && borders.is_contiguous(), name, ": borders int32 on the host");
  const Grad g = grad_of(name, dbias);
  const auto o = dbias.options().dtype(at::kFloat);
  const int64_t buckets = (nb + 1) * (both ? 2 : 1);
  if (!g.B || !g.Nq || !g.Nk) return at::zeros({buckets, g.H}, o);
  Tensor out = at::empty({buckets, g.H}, o);
  if (!on.meta) {
    const int H = small(name, g.H), Nq = small(name, g.Nq), Nk = small(name, g.Nk);
    Tensor ws = words(dbias, ovis_relpos_bias_1d_backward_workspace_bytes(g.B, H, Nq, Nk, (int)buckets));
    done(name, ovis_relpos_bias_1d_backward(dbias.const_data_ptr(), g.bs, g.hs, g.ld, out.data_ptr<float>(), ws.data_ptr<float>(), borders.const_data_ptr<int>(),
                                            nb, both, g.B, H, Nq, Nk, q_offset, d, cur_stream()));
  }
  return out;
}

Tensor swin_relpos_bias_backward(const Tensor& dbias, int64_t ws) {
  const char* name = "swin_relpos_bias_backward";
  On on(name, {&dbias});
  const int d = code(name, "dbias", dbias.scalar_type());
  TORCH_CHECK(ws >= 1 && ws <= 64, name, ": window size ", ws, " (1 to 64)");
  const Grad g = grad_of(name, dbias);
  TORCH_CHECK(g.Nq == ws * ws && g.Nk >= ws * ws, name, ": dbias must be [..., ", ws * ws, ", at least ", ws * ws, "], got ", dbias.sizes());
  const auto o = dbias.options().dtype(at::kFloat);
  const int64_t w = 2 * ws - 1;
  if (!g.B) return at::zeros({w * w, g.H}, o);
  Tensor out = at::empty({w * w, g.H}, o);
  if (!on.meta) {
    const int H = small(name, g.H);
    Tensor work = words(dbias, ovis_swin_relpos_bias_backward_workspace_bytes(g.B, H, (int)ws));
    done(name, ovis_swin_relpos_bias_backward(dbias.const_data_ptr(), g.bs, g.hs, g.ld, out.data_ptr<float>(), work.data_ptr<float>(), g.B, H, (int)ws, d,
                                              cur_stream()));
  }
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(ovis_mi, m) {
  m.def("layernorm_forward(Tensor x, Tensor gamma, Tensor beta, Tensor? residual, float eps, ScalarType? out_dtype, bool checkpoint) "
        "-> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("layernorm_backward(Tensor dy, Tensor? x, Tensor? codes, Tensor? scales, Tensor stats, Tensor gamma, Tensor? dsum, ScalarType? out_dtype) "
        "-> (Tensor, Tensor, Tensor)");
  m.def("act_forward_ckpt8(Tensor h, int act) -> (Tensor, Tensor, Tensor)");
  m.def("act_backward_ckpt8(Tensor dy, Tensor codes, Tensor scales, int act, bool recompute) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("ckpt8_decode(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor");
  m.def("linear_wgrad_ckpt8(Tensor dy, Tensor codes, Tensor scales, Tensor? gamma, Tensor? beta) -> (Tensor, Tensor)");
  m.def("relpos_bias_1d(Tensor table, Tensor borders, bool both, int Nq, int Nk, int q_offset, ScalarType dtype, int ld) -> Tensor");
  m.def("relpos_bias_1d_backward(Tensor dbias, Tensor borders, bool both, int q_offset) -> Tensor");
  m.def("swin_relpos_bias_backward(Tensor dbias, int ws) -> Tensor");
}
#define OVIS_TRAIN_OPS(m)                                            \
  m.impl("layernorm_forward", &layernorm_forward);                   \
  m.impl("layernorm_backward", &layernorm_backward);                 \
  m.impl("act_forward_ckpt8", &act_forward_ckpt8);                   \
  m.impl("act_backward_ckpt8", &act_backward_ckpt8);                 \
  m.impl("ckpt8_decode", &ckpt8_decode);                             \
  m.impl("linear_wgrad_ckpt8", &linear_wgrad_ckpt8);                 \
  m.impl("relpos_bias_1d", &relpos_bias_1d);                         \
  m.impl("relpos_bias_1d_backward", &relpos_bias_1d_backward);       \
  m.impl("swin_relpos_bias_backward", &swin_relpos_bias_backward);
TORCH_LIBRARY_IMPL(ovis_mi, CUDA, m) { OVIS_TRAIN_OPS(m) }           // "CUDA" is the HIP device's dispatch key on ROCm builds of torch
TORCH_LIBRARY_IMPL(ovis_mi, Meta, m) { OVIS_TRAIN_OPS(m) }
TORCH_LIBRARY_IMPL(ovis_mi, CPU, m) { OVIS_TRAIN_OPS(m) }            // refuses, with the reason
// they build no autograd graph, also where an argument requires a gradient (torch's own fallback would leave a node that warns)
TORCH_LIBRARY_IMPL(ovis_mi, Autograd, m) {
  for (const char* op : {"layernorm_forward", "layernorm_backward", "act_forward_ckpt8", "act_backward_ckpt8", "ckpt8_decode",
                         "linear_wgrad_ckpt8", "relpos_bias_1d", "relpos_bias_1d_backward", "swin_relpos_bias_backward"})
    m.impl(op, torch::CppFunction::makeFallthrough());
}
