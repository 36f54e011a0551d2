// The activation function of an MLP whose input h is kept in 8 bits for the backward pass (gfx950).
//
//   forward   y = act(h), h8 = the 8-bit form of h (train_elem.h)
//   backward  dh = dy * act'(h8), dbias = sum over rows dh, and if asked the 8-bit form of act(h8) (the operand of the next linear layer's
//             weight gradient, which then need not be kept either)
//
//   ReLU       act' = 1 where the code's sign bit is clear: the forward pass gives values that are not positive a set sign bit, so the
//              derivative is that of h itself even where its code underflows to 0 or h is -infinity (kept as -0; a NaN lets the gradient pass)
//   QuickGELU  act = h g, act' = g (1 + 1.702 h (1 - g)),  g = 1 / (1 + exp(-1.702 h))
//   GELU       act = h Phi, act' = Phi + h phi,  phi = exp(-h^2 / 2) / sqrt(2 pi), Phi = phi's integral
//
// Bound by HBM: h once, y and h8 once; dy and h8 once, dh once.  GELU's Phi is written over the exponential that phi needs anyway,
// Phi(-a) = exp(-a^2 / 2) t P(t) with t = 1 / (1 + 0.31 a), a >= 0: erfc's scaled form is smooth in t, and a polynomial of eight terms
// (least squares, reweighted towards the smallest relative error) is within 1.9e-7 of it up to a = 13.5, from where the exponential is no longer a
// normal f32 and becomes 0.  The exponential's argument is rounded, which adds 2^-24 of it: Phi(-a) in f32 is within 5e-7 of itself up to a = 1,
// 2e-6 up to 6, 8e-6 up to 13.
#include "train_elem.h"

namespace {

using namespace ovis;

constexpr float kLog2e = 1.4426950408889634f;

// exp(-a^2 / 2) and Phi(-a) for a = |h|
__device__ __forceinline__ void gauss(float h, float& e, float& tail) {
  const float a = fabsf(h);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.31f, a, 1.f));
  e = __builtin_amdgcn_exp2f(-0.5f * kLog2e * h * h);
  float p = 0.035840459f;
  p = fmaf(p, t, -0.14159951f);
  p = fmaf(p, t, 0.15505943f);
  p = fmaf(p, t, -0.014895893f);
  p = fmaf(p, t, 0.11010629f);
  p = fmaf(p, t, 0.10777222f);
  p = fmaf(p, t, 0.12406016f);
  p = fmaf(p, t, 0.12365692f);
  tail = p * t * e;
}

// act(h), and its derivative
template <int ACT>
__device__ __forceinline__ void activation(float h, float& y, float& slope) {
  if constexpr (ACT == 1) {
    y = h < 0.f ? 0.f : h;                                       // passes a NaN on
    slope = h == h && (__builtin_bit_cast(unsigned, h) >> 31) ? 0.f : 1.f;           // a decoded NaN has a sign of its own
  } else if constexpr (ACT == 2) {
    const float g = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.702f * kLog2e * h));
    y = h * g;
    slope = fmaf(1.702f, y * (1.f - g), g);                      // g (1 + 1.702 h (1 - g)), with no product above h
  } else if constexpr (ACT == 3) {
    float e, tail;
    gauss(h, e, tail);
    const float phi = h < 0.f ? tail : 1.f - tail;
    y = h * phi;
    slope = fmaf(h * 0.3989422804f, e, phi);
  } else {
    y = h;
    slope = 1.f;
  }
}

// a lane takes 8 columns of a row; the lanes of a row are padded to whole blocks of 32 columns, so that a block's four lanes are neighbours
template <typename T, int ACT>
__global__ void __launch_bounds__(256)
act_ckpt8_fwd_kernel(const T* __restrict__ h, long long ldh, T* __restrict__ y, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                     unsigned slots, unsigned per_row, long long rows, int C) {
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  if (i >= slots) return;                                        // slots is a multiple of 4: a block's lanes leave together
  const unsigned row = i / per_row, v = i - row * per_row;
  const int col = (int)v * 8, n = C - col;
  float x[8];
  if (n > 0) {
    load8(h + (long long)row * ldh + col, n, (long long)row + 8 < rows, x);          // eight rows on, a row's end is not the tensor's
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
  }
  unsigned sb;
  const u32x2_u q = encode8(x, ACT == 1, sb);
  if (n <= 0) return;
  const long long o = (long long)row * C + col;
  store_codes(codes + o, n, q);
  if ((v & 3) == 0) scales[(long long)row * (per_row >> 2) + (v >> 2)] = (uint8_t)sb;
  if constexpr (ACT != 0) {
    float s;
#pragma unroll
    for (int e = 0; e < 8; ++e) activation<ACT>(x[e], x[e], s);
    store8(y + o, n, x);
  }
}

// A workgroup owns a strip of 8 L columns and a run of rows, 256 / L of them at a time, so that a lane keeps the bias gradient of its eight
// columns in registers; L = 64, or the next power of two where a row is shorter.  The next row is fetched while the present one is worked on, and
// there are as many workgroups as the card holds.  73600 x 1536 fp16 GELU with the activation in 8 bits: 152 us, 4.5 TB/s (177 us without
// either; factor and slope from an LDS table over the 512 values that codes can stand for: 162 us).
template <typename T, int ACT>
__global__ void __launch_bounds__(256, 6)
act_ckpt8_bwd_kernel(const T* __restrict__ dy, long long lddy, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                     T* __restrict__ dh, uint8_t* __restrict__ codes2, uint8_t* __restrict__ scales2, float* __restrict__ part, long long rows,
                     long long chunk, int lshift, int C) {
  __shared__ float buf[256][9];
  const int L = 1 << lshift, li = threadIdx.x & (L - 1), ri = threadIdx.x >> lshift, rp = 256 >> lshift;
  const int v = (int)blockIdx.x * L + li, col = v * 8, n = C - col, nblk = (C + 31) >> 5;
  const bool mine = n > 0;
  const long long r0 = (long long)blockIdx.y * chunk, r1 = r0 + chunk < rows ? r0 + chunk : rows;
  float acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  Raw8<T> dn;                                                    // the next pass's row, fetched while the present one is worked on
  u32x2_u qn;
  unsigned sn;
  auto fetch = [&](long long r) {
    const int m = r < r1 ? n : 0;
    const bool on = r + 8 < rows;                                // eight rows on, a row's end is not the tensor's
    dn.load(dy + r * lddy + col, m, on);
    qn = load_codes(codes + r * C + col, m, on);
    sn = m > 0 ? scales[r * nblk + (col >> 5)] : 127u;
  };
  fetch(r0 + ri);
  for (long long rb = r0; rb < r1; rb += rp) {
    const long long r = rb + ri;
    const bool live = r < r1 && mine;
    const Raw8<T> raw = dn;
    const u32x2_u q = qn;
    const unsigned sb0 = sn;
    if (rb + rp < r1) fetch(r + rp);
    float h[8], d[8];
    decode8(q, sb0, h);                                          // behind the row's end: values that are neither stored nor summed up
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = raw.at(e);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float s;
      activation<ACT>(h[e], h[e], s);
      d[e] *= s;
      acc[e] += d[e];
    }
    if (live) store8(dh + r * C + col, n, d);
    if (codes2) {
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = e < n ? h[e] : 0.f;
      unsigned sb;
      const u32x2_u q = encode8(h, false, sb);
      if (live) {
        store_codes(codes2 + r * C + col, n, q);
        if ((v & 3) == 0) scales2[r * nblk + (col >> 5)] = (uint8_t)sb;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) buf[threadIdx.x][e] = acc[e];
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * L; i += 256) {
    const int c = (int)blockIdx.x * 8 * L + i;
    if (c < C) {
      float s = 0.f;
      for (int k = 0; k < rp; ++k) s += buf[k * L + (i >> 3)][i & 7];
      part[(long long)blockIdx.y * C + c] = s;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
ckpt8_decode_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out, unsigned slots, unsigned per_row,
                    int C) {
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  if (i >= slots) return;
  const unsigned row = i / per_row, v = i - row * per_row;
  const int col = (int)v * 8, n = C - col;
  float x[8];
  const long long o = (long long)row * C + col;
  decode8(load_codes(codes + o, n), scales[(long long)row * ((C + 31) >> 5) + (col >> 5)], x);
  store8(out + o, n, x);
}

struct BwdShape { int lshift; unsigned strips, chunks; long long chunk; };
inline BwdShape bwd_shape(long long rows, int C) {
  const int slots = (C + 31) / 32 * 4;
  BwdShape s;
  s.lshift = 2;
  while (s.lshift < 6 && (1 << s.lshift) < slots) ++s.lshift;
  s.strips = (unsigned)((slots + (1 << s.lshift) - 1) >> s.lshift);
  const int rp = 256 >> s.lshift;
  const long long most = (rows + rp - 1) / rp;                   // at least one pass of rows a workgroup
  long long want = s.strips < 1536 ? 1536 / s.strips : 1;        // six workgroups a CU in all: what is there at once
  if (want > most) want = most;
  if (most <= 4) want = 1;                                       // and no second launch: the workgroup's sums are the gradient
  s.chunk = ((rows + want - 1) / want + rp - 1) / rp * rp;
  s.chunks = (unsigned)((rows + s.chunk - 1) / s.chunk);
  return s;
}

}  // namespace

#define ACT_TYPE(dtype, CALL)                        \
  if (dtype == OVIS_F32) { CALL(float) }             \
  else if (dtype == OVIS_F16) { CALL(_Float16) }     \
  else { CALL(__bf16) }

extern "C" int ovis_act_ckpt8_forward(const void* h, long long ldh, void* y, uint8_t* codes, uint8_t* scales, long long rows, int C, int act,
                                      int dtype, ovis_stream_t stream) {
  OVIS_REQUIRE(h && codes && scales && (!y == !act), "act_ckpt8_forward: null pointer (y goes with an activation)");
  OVIS_REQUIRE(act >= 0 && act <= 3 && ovis::dtype_ok(dtype), "act_ckpt8_forward: activation %d, type %d", act, dtype);
  OVIS_REQUIRE(rows > 0 && C > 0 && ldh >= C, "act_ckpt8_forward: rows %lld, columns %d, row stride %lld", rows, C, ldh);
  const long long per_row = ((long long)C + 31) / 32 * 4;
  OVIS_REQUIRE(C <= (1 << 30) && rows <= 0xffffff00ll / per_row, "act_ckpt8_forward: %lld x %d is too large for one call", rows, C);
  const unsigned slots = (unsigned)(rows * per_row);
#define ACT_GO(T, A)                                                                                                                        \
  hipLaunchKernelGGL((act_ckpt8_fwd_kernel<T, A>), dim3(ovis::cdiv(slots, 256)), dim3(256), 0, (hipStream_t)stream, (const T*)h, ldh,      \
                     (T*)y, codes, scales, slots, (unsigned)per_row, rows, C)
#define ACT_ALL(T) switch (act) { case 0: ACT_GO(T, 0); break; case 1: ACT_GO(T, 1); break; case 2: ACT_GO(T, 2); break; default: ACT_GO(T, 3); }
  ACT_TYPE(dtype, ACT_ALL)
#undef ACT_GO
#undef ACT_ALL
  return ovis::check_launch("act_ckpt8_forward");
}

extern "C" long long ovis_act_ckpt8_backward_workspace_bytes(long long rows, int C) {
  if (rows <= 0 || C <= 0) return 0;
  return (long long)bwd_shape(rows, C).chunks * C * 4;
}

extern "C" int ovis_act_ckpt8_backward(const void* dy, long long lddy, const uint8_t* codes, const uint8_t* scales, void* dh, float* dbias,
                                       uint8_t* codes_out, uint8_t* scales_out, float* workspace, long long rows, int C, int act, int dtype,
                                       ovis_stream_t stream) {
  OVIS_REQUIRE(dy && codes && scales && dh && dbias && workspace && (!codes_out == !scales_out), "act_ckpt8_backward: null pointer");
  OVIS_REQUIRE(act >= 1 && act <= 3 && ovis::dtype_ok(dtype), "act_ckpt8_backward: activation %d, type %d", act, dtype);
  OVIS_REQUIRE(rows > 0 && C > 0 && C <= (1 << 30) && lddy >= C, "act_ckpt8_backward: rows %lld, columns %d, row stride %lld", rows, C, lddy);
  const BwdShape s = bwd_shape(rows, C);
  OVIS_REQUIRE(s.chunks <= 65535, "act_ckpt8_backward: too many rows for one launch");
  float* to = s.chunks == 1 ? dbias : workspace;
#define ACT_GO(T, A)                                                                                                                        \
  hipLaunchKernelGGL((act_ckpt8_bwd_kernel<T, A>), dim3(s.strips, s.chunks), dim3(256), 0, (hipStream_t)stream, (const T*)dy, lddy, codes, \
                     scales, (T*)dh, codes_out, scales_out, to, rows, s.chunk, s.lshift, C)
#define ACT_ALL(T) switch (act) { case 1: ACT_GO(T, 1); break; case 2: ACT_GO(T, 2); break; default: ACT_GO(T, 3); }
  ACT_TYPE(dtype, ACT_ALL)
#undef ACT_GO
#undef ACT_ALL
  const int rc = ovis::check_launch("act_ckpt8_backward");
  if (rc != OVIS_OK || s.chunks == 1) return rc;
  return ovis::column_sum_finish(workspace, (int)s.chunks, C, dbias, C, dbias, (hipStream_t)stream);
}

extern "C" int ovis_ckpt8_decode(const uint8_t* codes, const uint8_t* scales, void* out, long long rows, int C, int dtype, ovis_stream_t stream) {
  OVIS_REQUIRE(codes && scales && out && ovis::dtype_ok(dtype), "ckpt8_decode: null pointer or type %d", dtype);
  OVIS_REQUIRE(rows > 0 && C > 0, "ckpt8_decode: rows %lld, columns %d", rows, C);
  const long long per_row = ((long long)C + 7) / 8;
  OVIS_REQUIRE(C <= (1 << 30) && rows <= 0xffffff00ll / per_row, "ckpt8_decode: %lld x %d is too large for one call", rows, C);
  const unsigned slots = (unsigned)(rows * per_row);
#define DEC_ALL(T)                                                                                                                          \
  hipLaunchKernelGGL((ckpt8_decode_kernel<T>), dim3(ovis::cdiv(slots, 256)), dim3(256), 0, (hipStream_t)stream, codes, scales, (T*)out,    \
                     slots, (unsigned)per_row, C);
  ACT_TYPE(dtype, DEC_ALL)
#undef DEC_ALL
  return ovis::check_launch("ckpt8_decode");
}
