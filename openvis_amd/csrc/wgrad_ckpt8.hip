// Weight gradient of a linear layer from its input in 8 bits (gfx950):
//
//   dW[n, k] = sum over m dY[m, n] X[m, k],  db[n] = sum over m dY[m, n],  X = the values of the e4m3 codes (train_elem.h)
//   with gamma, beta: X stands for a layer norm's normalised rows, the layer's input was X gamma + beta:
//   dW[n, k] = gamma[k] sum dY X + beta[k] db[n]
//
// Bound by the matrix cores (2 M N K flop) when N and K are large.  Both operands lie with the summed dimension m along their rows, so a tile
// of BM rows of each is laid row by row into LDS and the fragments, 8 consecutive m of one column a lane, come out through the transposing
// LDS read.  X is widened while it is staged, where 32 neighbouring columns share a scale: to bf16 (4 significant bits and any scale: exact).
//   dY bf16: one bf16 product.  dY f32: three (f32 = the sum of three bf16 numbers), f32-grade.
//   dY fp16: fp16 products; X is scaled per 32 columns by the largest scale of the workgroup's rows so that its largest code comes to at most
//   57344: exact for scales down to 2^-22 of the largest, below that off by at most 2^-30 of the 32 columns' largest value.
// All products are exact in f32; sums are f32.  Rows are split over workgroups (S parts) where there are too few tiles to fill the card; the
// parts are added in a fixed order by a second kernel.
#include "train_elem.h"

namespace {

using namespace ovis;

using f32x16 = __attribute__((ext_vector_type(16))) float;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using u16x8 = __attribute__((ext_vector_type(8))) unsigned short;
using u16x4 = __attribute__((ext_vector_type(4))) unsigned short;
using f16x2 = __attribute__((ext_vector_type(2))) _Float16;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
typedef short s16x4 __attribute__((__vector_size__(4 * sizeof(short))));

// 16 lanes read 4 rows of 16 columns and get one column's 4 rows each
__device__ __forceinline__ u16x4 tr_read(const unsigned short* p) {
  const s16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(const_cast<unsigned short*>(p)));
  return __builtin_bit_cast(u16x4, r);
}

template <bool F16>
__device__ __forceinline__ f32x16 mfma(u16x8 a, u16x8 b, f32x16 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// an LDS tile [rows][W] of 16-bit elements; the 32-column pieces of a row are permuted by the row, so that the four rows of a transposing
// read lie in different banks
template <int W>
__device__ __forceinline__ int at(int m, int c) {
  const int s = W >= 128 ? m & 3 : (m >> 1) & 1;
  return m * W + ((((c >> 5) ^ s) << 5) | (c & 31));
}

template <typename T> struct DyOf {                              // 8 elements of dY as loaded
  u16x8 v;
  __device__ __forceinline__ void load(const T* __restrict__ p, int n) {
    if (n >= 8) {
      v = __builtin_bit_cast(u16x8, *reinterpret_cast<const typename Vec8Of<T>::type*>(p));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < n ? __builtin_bit_cast(unsigned short, p[e]) : (unsigned short)0;
    }
  }
  __device__ __forceinline__ void load_all(const T* __restrict__ p) {
    v = __builtin_bit_cast(u16x8, *reinterpret_cast<const typename Vec8Of<T>::type*>(p));
  }
  __device__ __forceinline__ float value(int e) const { return (float)__builtin_bit_cast(T, (unsigned short)v[e]); }
  __device__ __forceinline__ u16x8 plane(int) const { return v; }
};
template <> struct DyOf<float> {
  float v[8];
  __device__ __forceinline__ void load(const float* __restrict__ p, int n) { load8(p, n, v); }
  __device__ __forceinline__ void load_all(const float* __restrict__ p) { load8(p, 8, v); }
  __device__ __forceinline__ float value(int e) const { return v[e]; }
  __device__ __forceinline__ u16x8 plane(int i) const {         // the i-th bf16 term of v (each the rest rounded to nearest)
    u16x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x = v[e];
      __bf16 t = (__bf16)x;
      if (i > 0) { x -= (float)t; t = (__bf16)x; }
      if (i > 1) { x -= (float)t; t = (__bf16)x; }
      r[e] = __builtin_bit_cast(unsigned short, t);
    }
    return r;
  }
};

template <bool F16>
__device__ __forceinline__ u16x8 widen(u32x2_u c, float f) {
  unsigned r[4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (F16) {
      r[2 * h] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[h], f, false));
      r[2 * h + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[h], f, true));
    } else {
      r[2 * h] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[h], f, false));
      r[2 * h + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[h], f, true));
    }
  }
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  u32x4 q = {r[0], r[1], r[2], r[3]};
  return __builtin_bit_cast(u16x8, q);
}

// TN x TK: the workgroup's tile of dW; WN x WK wavefronts; BM rows a step
template <typename T, int TN, int TK, int WN, int WK, int BM>
__global__ void __launch_bounds__(64 * WN * WK)
wgrad_ckpt8_kernel(const T* __restrict__ dy, long long lddy, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                   float* __restrict__ out, float* __restrict__ dbp, long long M, int N, int K, long long chunk, int tiles_n, int tiles_k) {
  constexpr bool F16 = sizeof(T) == 2 && !__is_same(T, __bf16);
  constexpr int P = sizeof(T) == 4 ? 3 : 1, NT = 64 * WN * WK, RN = TN / WN, RK = TK / WK, AN = RN / 32, AK = RK / 32;
  constexpr int YR = NT / (TN / 8), XR = NT / (TK / 8), YP = BM / YR, XP = BM / XR;        // rows a pass, passes
  extern __shared__ unsigned short lds[];
  unsigned short* ly = lds;                                      // [2][P][BM][TN]
  unsigned short* lx = lds + 2 * P * BM * TN;                    // [2][BM][TK]
  __shared__ int top[TK / 32];
  const unsigned id = xcd_remap(blockIdx.x, gridDim.x);          // an XCD's workgroups: neighbouring tiles of the same rows
  const int nt = id % tiles_n, kt = (id / tiles_n) % tiles_k;
  const long long s = id / (tiles_n * tiles_k);
  const long long m0 = s * chunk, m1 = m0 + chunk < M ? m0 + chunk : M;
  const int n0 = nt * TN, k0 = kt * TK, nblk = (K + 31) >> 5;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wn = wave / WK, wk = wave % WK;

  if constexpr (F16) {                                           // the largest scale of each 32 columns over the workgroup's rows
    if (tid < TK / 32) top[tid] = 0;
    __syncthreads();
    const int b0 = k0 >> 5, nb = min(TK / 32, nblk - b0);
    const int b = tid % (TK / 32);
    int t = 0;
    if (b < nb)
      for (long long m = m0 + tid / (TK / 32); m < m1; m += NT / (TK / 32)) t = max(t, (int)scales[m * nblk + b0 + b]);
    atomicMax(&top[b], t);                                       // a maximum: the order does not matter
    __syncthreads();
  }

  const int yr = tid / (TN / 8), yc = (tid % (TN / 8)) * 8, xr = tid / (TK / 8), xc = (tid % (TK / 8)) * 8;
  const int yn = N - n0 - yc, xn = K - k0 - xc;
  const int xtop = F16 ? top[xc >> 5] - 7 : 0;
  DyOf<T> ry[YP];
  u32x2_u rx[XP];
  unsigned rs[XP];
  const bool whole = n0 + TN <= N && k0 + TK <= K;               // no column of the tile lies outside
  auto fetch = [&](long long m) {
    if (whole && m + BM <= m1) {
      const T* py = dy + (m + yr) * lddy + n0 + yc;
      const uint8_t* pc = codes + (m + xr) * K + k0 + xc;
      const uint8_t* ps = scales + (m + xr) * nblk + ((k0 + xc) >> 5);
#pragma unroll
      for (int i = 0; i < YP; ++i) ry[i].load_all(py + (long long)i * YR * lddy);
#pragma unroll
      for (int i = 0; i < XP; ++i) {
        rx[i] = *reinterpret_cast<const u32x2_u*>(pc + (long long)i * XR * K);
        rs[i] = ps[(long long)i * XR * nblk];
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < YP; ++i) {
      const long long r = m + yr + i * YR;
      ry[i].load(dy + (r < m1 ? r : m1 - 1) * lddy + n0 + (yn > 0 ? yc : 0), r < m1 ? yn : 0);
    }
#pragma unroll
    for (int i = 0; i < XP; ++i) {
      const long long r = m + xr + i * XR;
      const bool ok = r < m1 && xn > 0;
      rx[i][0] = rx[i][1] = 0u;
      rs[i] = 127u;
      if (ok) {
        rx[i] = load_codes(codes + r * K + k0 + xc, xn);
        rs[i] = scales[r * nblk + ((k0 + xc) >> 5)];
      }
    }
  };
  float dsum[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dsum[e] = 0.f;
  auto stage = [&](int buf) {
#pragma unroll
    for (int i = 0; i < YP; ++i) {
#pragma unroll
      for (int p = 0; p < P; ++p)
        *reinterpret_cast<u16x8*>(ly + (buf * P + p) * BM * TN + at<TN>(yr + i * YR, yc)) = ry[i].plane(p);
      if (kt == 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) dsum[e] += ry[i].value(e);
      }
    }
#pragma unroll
    for (int i = 0; i < XP; ++i) {
      const int e = F16 ? max((int)rs[i] - xtop, -60) : (int)rs[i] - 127;      // 60 octaves below the largest nothing is left in fp16
      *reinterpret_cast<u16x8*>(lx + buf * BM * TK + at<TK>(xr + i * XR, xc)) = widen<F16>(rx[i], pow2f(e));
    }
  };

  f32x16 acc[AN][AK];
#pragma unroll
  for (int a = 0; a < AN; ++a)
#pragma unroll
    for (int b = 0; b < AK; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;

  const int li = lane & 15, half = lane >> 5, colg = 16 * ((lane >> 4) & 1) + 4 * (li & 3), rowg = 8 * half + (li >> 2);
  fetch(m0);
  stage(0);
  fetch(m0 + BM);
  __syncthreads();
  int buf = 0;
  for (long long m = m0; m < m1; m += BM) {
    const unsigned short* py = ly + buf * P * BM * TN;
    const unsigned short* px = lx + buf * BM * TK;
#pragma unroll
    for (int st = 0; st < BM / 16; ++st) {
      if (st == BM / 32) {                                       // halfway: the next rows into the other buffer, the ones behind them from memory
        if (m + BM < m1) stage(buf ^ 1);
        if (m + 2 * BM < m1) fetch(m + 2 * BM);
      }
      u16x8 fb[AK];
#pragma unroll
      for (int b = 0; b < AK; ++b) {
        const u16x4 u = tr_read(px + at<TK>(16 * st + rowg, wk * RK + b * 32 + colg)), v = tr_read(px + at<TK>(16 * st + rowg + 4, wk * RK + b * 32 + colg));
        fb[b] = __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
      }
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int a = 0; a < AN; ++a) {
          const unsigned short* q = py + p * BM * TN;
          const u16x4 u = tr_read(q + at<TN>(16 * st + rowg, wn * RN + a * 32 + colg)), v = tr_read(q + at<TN>(16 * st + rowg + 4, wn * RN + a * 32 + colg));
          const u16x8 fa = __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
          for (int b = 0; b < AK; ++b) acc[a][b] = mfma<F16>(fa, fb[b], acc[a][b]);
        }
    }
    __syncthreads();
    buf ^= 1;
  }

  // a lane holds column k = lane & 31 of its blocks; register r is row (r & 3) + 8 (r >> 2) + 4 half
  float* o = out + s * N * K;
#pragma unroll
  for (int b = 0; b < AK; ++b) {
    const int kl = wk * RK + b * 32, k = k0 + kl + (lane & 31);
    const float f = F16 ? pow2f(top[kl >> 5] - 127 - 7) : 1.f;
    if (k < K) {
#pragma unroll
      for (int a = 0; a < AN; ++a)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int n = n0 + wn * RN + a * 32 + (r & 3) + 8 * (r >> 2) + 4 * half;
          if (n < N) o[(long long)n * K + k] = acc[a][b][r] * f;
        }
    }
  }
  if (kt == 0) {                                                 // db: the lanes of a column group, in order
    float* sum = reinterpret_cast<float*>(lds);                  // [YR][TN]
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[yr * TN + yc + e] = dsum[e];
    __syncthreads();
    for (int c = tid; c < TN; c += NT) {
      float t = 0.f;
      for (int i = 0; i < YR; ++i) t += sum[i * TN + c];
      if (n0 + c < N) dbp[s * N + n0 + c] = t;
    }
  }
}

// dw = gamma sum over the parts + beta db
__global__ void __launch_bounds__(256)
wgrad_join_kernel(const float* __restrict__ part, int S, const float* __restrict__ db, const float* __restrict__ gamma, const float* __restrict__ beta,
                  float* __restrict__ dw, long long NK, int K) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= NK) return;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  const int n = NK - i < 4 ? (int)(NK - i) : 4;
  typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
  for (int s = 0; s < S; ++s) {
    const float* p = part + s * NK + i;
    if (n == 4) {
      const f32x4_u t = *reinterpret_cast<const f32x4_u*>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += t[e];
    } else {
      for (int e = 0; e < n; ++e) v[e] += p[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (e < n) {
      float t = v[e];
      if (gamma) {
        const long long r = (i + e) / K;
        const int k = (int)(i + e - r * K);
        t = t * gamma[k] + beta[k] * db[r];
      }
      dw[i + e] = t;
    }
  }
}

struct WgradShape { int tile, tiles_n, tiles_k, S; long long chunk; };
inline WgradShape wgrad_shape(long long M, int N, int K, int dtype) {
  WgradShape w;
  const long long t256 = (long long)cdiv(N, 256) * cdiv(K, 256), t128 = (long long)cdiv(N, 128) * cdiv(K, 128);
  w.tile = dtype != OVIS_F32 && t256 * ((M + 1023) / 1024) >= 256 ? 256 : t128 * ((M + 511) / 512) >= 256 ? 128 : 64;
  w.tiles_n = (int)cdiv(N, w.tile);
  w.tiles_k = (int)cdiv(K, w.tile);
  const long long tiles = (long long)w.tiles_n * w.tiles_k, slots = w.tile == 256 ? 256 : 512;
  long long S = tiles >= slots ? 1 : slots / tiles;
  const long long most = (M + 255) / 256;                        // 256 rows at least
  if (S > most) S = most;
  w.chunk = ((M + S - 1) / S + 63) / 64 * 64;
  w.S = (int)((M + w.chunk - 1) / w.chunk);
  return w;
}

}  // namespace

extern "C" long long ovis_linear_wgrad_ckpt8_workspace_bytes(long long M, int N, int K, int dtype) {
  if (M <= 0 || N <= 0 || K <= 0 || !ovis::dtype_ok(dtype)) return 0;
  const WgradShape w = wgrad_shape(M, N, K, dtype);
  return ((long long)w.S * N * K + (long long)w.S * N) * 4;
}

extern "C" int ovis_linear_wgrad_ckpt8(const void* dy, long long lddy, const uint8_t* codes, const uint8_t* scales, const float* gamma,
                                       const float* beta, float* dw, float* db, float* workspace, long long M, int N, int K, int dtype,
                                       ovis_stream_t stream) {
  OVIS_REQUIRE(dy && codes && scales && dw && db && workspace && (!gamma == !beta), "linear_wgrad_ckpt8: null pointer");
  OVIS_REQUIRE(M > 0 && N > 0 && K > 0 && lddy >= N && ovis::dtype_ok(dtype), "linear_wgrad_ckpt8: M %lld, N %d, K %d, row stride %lld, type %d", M, N,
               K, lddy, dtype);
  const WgradShape w = wgrad_shape(M, N, K, dtype);
  const long long blocks = (long long)w.tiles_n * w.tiles_k * w.S;
  OVIS_REQUIRE(blocks < (1ll << 31) && (long long)N * K < (1ll << 40), "linear_wgrad_ckpt8: %d x %d is too large for one call", N, K);
  const bool join = w.S > 1 || gamma;
  float* part = join ? workspace : dw;
  float* dbp = w.S > 1 ? workspace + (long long)w.S * N * K : db;
#define WG_GO(T, TN, TK, WN, WK, BM)                                                                                                        \
  {                                                                                                                                         \
    const int lds = 2 * BM * (TN * (sizeof(T) == 4 ? 3 : 1) + TK) * 2;                                                                      \
    const hipError_t e = hipFuncSetAttribute((const void*)wgrad_ckpt8_kernel<T, TN, TK, WN, WK, BM>,                                        \
                                             hipFuncAttributeMaxDynamicSharedMemorySize, lds);                                              \
    OVIS_REQUIRE(e == hipSuccess, "linear_wgrad_ckpt8: %s", hipGetErrorString(e));                                                          \
    hipLaunchKernelGGL((wgrad_ckpt8_kernel<T, TN, TK, WN, WK, BM>), dim3((unsigned)blocks), dim3(64 * WN * WK), lds, (hipStream_t)stream,   \
                       (const T*)dy, lddy, codes, scales, part, dbp, M, N, K, w.chunk, w.tiles_n, w.tiles_k);                               \
  }
  if (dtype == OVIS_F32) {
    if (w.tile == 128) WG_GO(float, 128, 128, 2, 2, 32)
    else WG_GO(float, 64, 64, 2, 2, 32)
  } else if (dtype == OVIS_F16) {
    if (w.tile == 256) WG_GO(_Float16, 256, 256, 2, 4, 64)
    else if (w.tile == 128) WG_GO(_Float16, 128, 128, 2, 2, 64)
    else WG_GO(_Float16, 64, 64, 2, 2, 64)
  } else {
    if (w.tile == 256) WG_GO(__bf16, 256, 256, 2, 4, 64)
    else if (w.tile == 128) WG_GO(__bf16, 128, 128, 2, 2, 64)
    else WG_GO(__bf16, 64, 64, 2, 2, 64)
  }
#undef WG_GO
  int rc = ovis::check_launch("linear_wgrad_ckpt8");
  if (rc == OVIS_OK && w.S > 1) rc = ovis::column_sum_finish(dbp, w.S, N, db, N, db, (hipStream_t)stream);
  if (rc != OVIS_OK || !join) return rc;
  const long long NK = (long long)N * K;
  hipLaunchKernelGGL(wgrad_join_kernel, dim3(ovis::cdiv((NK + 3) / 4, 256)), dim3(256), 0, (hipStream_t)stream, part, w.S, db, gamma, beta, dw, NK, K);
  return ovis::check_launch("linear_wgrad_ckpt8");
}
