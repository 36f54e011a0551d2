// Weight gradient of a linear layer from its input in 8 bits (gfx950):
//
//   dW[n, k] = sum over m dY[m, n] X[m, k],  db[n] = sum over m dY[m, n],  X = the values of the e4m3 codes (train_elem.h)
//   with gamma, beta: X stands for a layer norm's normalised rows, the layer's input was X gamma + beta:
//   dW[n, k] = gamma[k] sum dY X + beta[k] db[n]
//
// Bound by the matrix cores (2 M N K flop) when N and K are large.  Both operands lie with the summed dimension m along their rows, so a tile
// of BM rows of each is laid row by row into LDS and the fragments, 8 consecutive m of one column a lane, come out through the transposing
// LDS read.  X is widened while it is staged, where 32 neighbouring columns share a scale: to bf16 (4 significant bits and any scale: exact).
//   dY bf16: one bf16 product.  dY f32: three (f32 = the sum of three bf16 numbers, exact for magnitudes from 2^-110 on; smaller ones are off by
//   at most 2^-133, bf16's last bit; an infinity minus itself makes its column's sums NaN).
//   dY fp16: fp16 products; X is scaled per 32 columns by the largest scale of the workgroup's rows so that its largest code comes to at most
//   57344: exact for scales down to 2^-22 of the largest.  A workgroup that meets a smaller one (rows far apart in size, the large ones perhaps
//   with no gradient at all) throws its sums away and takes its rows again with dY as the sum of two bf16 numbers (11 bits: exact), which
//   takes about four times as long.  Blocks of the format's smallest scale, 2^-100, do not count: they are the zeros of padding and of ReLU; what
//   values they hold, below 2^-91, are taken as 0 where the 32 columns' largest scale is 2^-77 or more.
// All products are exact in f32; sums are f32.  Rows are split over workgroups (S parts) where there are too few tiles to fill the card; the
// parts are added in a fixed order by a second kernel.  36928 x 1024 x 4096 fp16: 270 to 284 us by the card, 1.09 to
// 1.15 PFLOP/s (2000 x 1000 x 1000: 24 us).
#include "train_elem.h"
#include <type_traits>

namespace {

using namespace ovis;

typedef unsigned u32_u __attribute__((aligned(1)));
typedef unsigned short u16_u __attribute__((aligned(1)));
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
// read lie in different banks, and of 256 columns the upper ones have the halves of a piece exchanged, so that eight lanes that write a
// piece each (X's codes) do too
template <int W>
__device__ __forceinline__ int at(int m, int c) {
  const int s = W >= 128 ? m & 3 : (m >> 1) & 1, x = W == 256 ? (c >> 3) & 16 : 0;
  return m * W + ((((c >> 5) ^ s) << 5) | ((c & 31) ^ x));
}

template <typename T> struct DyOf {                              // 8 elements of dY as loaded
  u16x8 v;
  __device__ __forceinline__ void load(const T* p, int n) {      // n <= 0: none
    v = (u16x8)0;
    if (n >= 8) {
      load_all(p);
    } else if (n > 0) {
      T t[7];
#pragma unroll
      for (int e = 0; e < 7; ++e) t[e] = p[e < n ? e : n - 1];
#pragma unroll
      for (int e = 0; e < 7; ++e) v[e] = e < n ? __builtin_bit_cast(unsigned short, t[e]) : (unsigned short)0;
    }
  }
  __device__ __forceinline__ void load_all(const T* p) { v = __builtin_bit_cast(u16x8, *reinterpret_cast<const typename Vec8Of<T>::type*>(p)); }
  __device__ __forceinline__ float value(int e) const { return (float)__builtin_bit_cast(T, (unsigned short)v[e]); }
  __device__ __forceinline__ u16x8 plane(int) const { return v; }
};
template <> struct DyOf<float> {
  float v[8];
  __device__ __forceinline__ void load(const float* p, int n) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (n > 0) load8(p, n, v);
  }
  __device__ __forceinline__ void load_all(const float* p) { load8(p, 8, v); }
  __device__ __forceinline__ float value(int e) const { return v[e]; }
  // the i-th bf16 term of v, each the upper half of what is left: 8 of the 24 significant bits, so that the three are exact and none is larger than v
  // (rounded to nearest the first term of values from 2^128 (1 - 2^-9) on would be an infinity)
  __device__ __forceinline__ u16x8 plane(int i) const {
    u16x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x = v[e];
#pragma unroll
      for (int k = 0; k < i; ++k) x -= __builtin_bit_cast(float, __builtin_bit_cast(unsigned, x) & 0xffff0000u);
      r[e] = (unsigned short)(__builtin_bit_cast(unsigned, x) >> 16);
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

// TN x TK: the workgroup's tile of dW, on WN x WK wavefronts; BM rows a step.
//
// The K loop.  LDS holds three steps: one that is multiplied, the next (its first fragments are read while the last products of the present
// one run), and one that is being written; so a step needs one barrier, and nothing waits behind it.  Registers hold three more steps on
// their way from memory.  A step's rows are fetched without a mask: a lane whose columns lie outside the matrix reads the first ones (its products
// go to rows or columns of dW that are not written), and one whose eight columns cross the row's end reads on into the next row; the rows
// for which that would leave the matrix, the last ones, are done behind the loop with masks.
template <typename T, int TN, int TK, int WN, int WK, int BM>
__global__ void __launch_bounds__(64 * WN * WK)
wgrad_ckpt8_kernel(const T* __restrict__ dy, long long lddy, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                   float* __restrict__ out, float* __restrict__ dbp, long long M, int N, int K, long long chunk, int tiles_n, int tiles_k, int turns,
                   const uint8_t* __restrict__ tops, int tshift) {
  constexpr bool F16 = sizeof(T) == 2 && !__is_same(T, __bf16);
  constexpr int P = sizeof(T) == 4 ? 3 : 1, NT = 64 * WN * WK, RN = TN / WN, RK = TK / WK, AN = RN / 32, AK = RK / 32, NS = BM / 16;
  constexpr int YR = NT / (TN / 8), YP = BM / YR;                // dY: rows a pass, passes of eight columns a lane
  constexpr int XC = BM * TK / NT, XP = XC / 8;                  // X: columns a lane takes of one row, inside one block of 32: one scale
  static_assert(YP * YR == BM && YP > 0 && XC * NT == BM * TK && (XC == 8 || XC == 16 || XC == 32), "a step is whole passes");
  extern __shared__ unsigned short lds[];
  unsigned short* const ly = lds;                                // [3][P][BM][TN]
  unsigned short* const lx = lds + 3 * P * BM * TN;              // [3][BM][TK]
  __shared__ int top[TK / 32];
  const unsigned id = xcd_remap(blockIdx.x, gridDim.x);          // an XCD's workgroups: neighbouring tiles of the same rows
  const int nt = id % tiles_n, kt = (id / tiles_n) % tiles_k;
  const long long s = id / (tiles_n * tiles_k);
  const long long m0 = s * chunk, m1 = m0 + chunk < M ? m0 + chunk : M;
  const int n0 = nt * TN, k0 = kt * TK, nblk = (K + 31) >> 5;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wn = wave / WK, wk = wave % WK;

  if constexpr (F16) {                                           // the largest scale of each 32 columns over the workgroup's rows
    if (tid < TK / 32) top[tid] = 27;                           // the smallest scale that the 8-bit form has
    __syncthreads();
    // from the scales themselves, or from the largest of 32 rows each (tops, tshift 5).  A lane reads a row's TK / 32 bytes at once (those behind
    // the row's end belong to the next row, and to columns that are not used); the last rows, where that would leave the array, byte by byte
    typedef unsigned short pairs __attribute__((ext_vector_type(2)));
    constexpr int NB = TK / 32, NW = NB > 4 ? NB / 4 : 1;
    const int b0 = k0 >> 5;
    const long long up = (1ll << tshift) - 1, r0 = m0 >> tshift, r1 = (m1 + up) >> tshift, all = (M + up) >> tshift;
    const long long whole = all - 8 < r1 ? all - 8 : r1;
    pairs hi[NW][2];
#pragma unroll
    for (int w = 0; w < NW; ++w) hi[w][0] = hi[w][1] = (pairs)0;
#pragma unroll 8
    for (long long m = r0 + tid; m < whole; m += NT) {
      const uint8_t* p = tops + m * nblk + b0;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const unsigned v = NB >= 4 ? *reinterpret_cast<const u32_u*>(p + 4 * w) : *reinterpret_cast<const u16_u*>(p);
        hi[w][0] = __builtin_elementwise_max(hi[w][0], __builtin_bit_cast(pairs, v & 0x00ff00ffu));
        hi[w][1] = __builtin_elementwise_max(hi[w][1], __builtin_bit_cast(pairs, (v >> 8) & 0x00ff00ffu));
      }
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      int t = hi[i / 4][i & 1][(i >> 1) & 1];
      const long long m = (whole > r0 ? whole : r0) + tid;
      if (m < r1 && b0 + i < nblk) t = max(t, (int)tops[m * nblk + b0 + i]);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) t = max(t, __shfl_xor(t, o, 64));
      if (lane == 0) atomicMax(&top[i], t);                      // a maximum: the order does not matter
    }
    __syncthreads();
  }

  const int yr = tid / (TN / 8), yc = (tid % (TN / 8)) * 8, xr = tid / (TK / XC), xc = (tid % (TK / XC)) * XC;
  const int yn = N - n0 - yc, xn = K - k0 - xc;                  // columns from this lane's first on
  const int xtop = F16 ? top[xc >> 5] - 7 : 0;
  int lowest = 0;                                                // the smallest exponent that codes are widened with, blocks of the smallest scale aside
  struct Rows { DyOf<T> y[YP]; u32x2_u x[XP]; unsigned s; };
  // no masks; a step's uniform row pointers and a lane's 32-bit offsets from them; in pieces, to lie between the products
  struct At { const T* y; const uint8_t *c, *s; };
  const unsigned oy = yr * (unsigned)lddy + (yn > 0 ? n0 + yc : 0), oc = xr * (unsigned)K + (xn > 0 ? k0 + xc : 0);
  const unsigned os = xr * (unsigned)nblk + (xn > 0 ? (k0 + xc) >> 5 : 0);
  constexpr int XL = XC >= 16 ? XC / 16 : 1, NF = YP + XL + 1;   // loads of a lane's codes, of a step
  auto fetch_piece = [&](Rows& R, const At& p, int i) {
    if (i < YP) {
      R.y[i].load_all(p.y + (long long)(i * YR) * lddy + oy);
    } else if (i < YP + XL) {
      if constexpr (XC >= 16) {
        typedef unsigned u32x4_u __attribute__((ext_vector_type(4), aligned(1)));
        const int j = 2 * (i - YP);
        const u32x4_u c = *reinterpret_cast<const u32x4_u*>(p.c + 8 * j + oc);
        R.x[j] = __builtin_shufflevector(c, c, 0, 1), R.x[j + 1] = __builtin_shufflevector(c, c, 2, 3);
      } else {
        R.x[0] = *reinterpret_cast<const u32x2_u*>(p.c + oc);
      }
    } else {
      // with the three bytes behind it: a byte's load would be widened, and so waited for, a step before it is used
      R.s = *reinterpret_cast<const u32_u*>(p.s + os);
    }
  };
  auto fetch_masked = [&](Rows& R, long long m) {
#pragma unroll
    for (int i = 0; i < YP; ++i) {
      const long long r = m + yr + i * YR;
      R.y[i].load(dy + (r < m1 ? r : m1 - 1) * lddy + n0 + (yn > 0 ? yc : 0), r < m1 ? yn : 0);
    }
    const long long r = m + xr;
    const bool ok = r < m1 && xn > 0;
#pragma unroll
    for (int j = 0; j < XP; ++j) {
      const int n = ok ? xn - 8 * j : 0;
      R.x[j] = load_codes(codes + (n > 0 ? r * K + k0 + xc + 8 * j : 0), n);
    }
    R.s = ok ? scales[r * nblk + ((k0 + xc) >> 5)] : F16 ? (unsigned)xtop : 127u;
  };
  float dsum[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dsum[e] = 0.f;
  // db: every workgroup of these rows and columns n stages all of dY; the first `turns` of them take the steps in turn
  int turn = kt < turns ? kt : -1;
  auto sum_rows = [&](const Rows& R, bool valid) {
    if (turn == 0 && valid) {
#pragma unroll
      for (int i = 0; i < YP; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) dsum[e] += R.y[i].value(e);
    }
    turn = turn == 0 ? turns - 1 : turn < 0 ? -1 : turn - 1;
  };
  auto stage_piece = [&](const Rows& R, int buf, int i) {
    if (i < YP) {
#pragma unroll
      for (int p = 0; p < P; ++p)
        *reinterpret_cast<u16x8*>(ly + (buf * P + p) * BM * TN + at<TN>(yr + i * YR, yc)) = R.y[i].plane(p);
    } else {
      const int j = i - YP, sb = (int)(R.s & 0xffu), e = F16 ? max(sb - xtop, -60) : sb - 127;      // 60 octaves below the largest nothing is left in fp16
      if constexpr (F16) lowest = min(lowest, sb == 27 ? 0 : e);
      *reinterpret_cast<u16x8*>(lx + buf * BM * TK + at<TK>(xr, xc + 8 * j)) = widen<F16>(R.x[j], pow2f(e));
    }
  };

  f32x16 acc[AN][AK];
#pragma unroll
  for (int a = 0; a < AN; ++a)
#pragma unroll
    for (int b = 0; b < AK; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;

  struct Frags { u16x8 a[P][AN], b[AK]; };
  const int li = lane & 15, half = lane >> 5, colg = 16 * ((lane >> 4) & 1) + 4 * (li & 3), rowg = 8 * half + (li >> 2);
  // fragment i of a substep: first the ones of X, then those of dY
  auto read_piece = [&](Frags& F, int buf, int st, int i) {
    if (i < AK) {
      const unsigned short* q = lx + buf * BM * TK + 16 * st * TK + at<TK>(rowg, wk * RK + i * 32 + colg);
      F.b[i] = __builtin_shufflevector(tr_read(q), tr_read(q + 4 * TK), 0, 1, 2, 3, 4, 5, 6, 7);      // 4 rows on: the same permutation
    } else {
      const int p = (i - AK) / AN, a = (i - AK) % AN;
      const unsigned short* q = ly + (buf * P + p) * BM * TN + 16 * st * TN + at<TN>(rowg, wn * RN + a * 32 + colg);
      F.a[p][a] = __builtin_shufflevector(tr_read(q), tr_read(q + 4 * TN), 0, 1, 2, 3, 4, 5, 6, 7);
    }
  };
  constexpr int G = P * AN * AK, NR = AK + P * AN, NQ = YP + XP; // products a substep; its fragments; writes of a step's rows
  auto multiply = [&](const Frags& F, int g) {
    const int p = g / (AN * AK), a = g / AK % AN, b = g % AK;
    acc[a][b] = mfma<F16>(F.a[p][a], F.b[b], acc[a][b]);
  };

  // steps that need no mask: all their rows lie in the chunk, and what a lane reads behind a row's end lies in the matrix
  const long long mf = m1 > M - 8 ? (M - 8 > m0 ? M - 8 : m0) : m1;
  const long long nf = lddy < 8 || K < 8 ? 0 : (mf - m0) / BM;
  if (nf > 0) {
    Rows R[3];
    Frags F[2];
    At next = {dy + m0 * lddy, codes + m0 * K, scales + m0 * nblk};
    long long fetched = 0;                                       // a step of the last rows is fetched again rather than one behind them
    auto advance = [&]() {
      const bool more = ++fetched < nf;
      next.y += more ? BM * lddy : 0, next.c += more ? BM * (long long)K : 0, next.s += more ? BM * (long long)nblk : 0;
    };
#pragma unroll
    for (int u = 0; u < 5; ++u) {
      if (u > 2) {
        sum_rows(R[u - 3], u - 3 < nf);
#pragma unroll
        for (int i = 0; i < NQ; ++i) stage_piece(R[u - 3], u - 3, i);
      }
#pragma unroll
      for (int i = 0; i < NF; ++i) fetch_piece(R[u % 3], next, i);
      advance();
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NR; ++i) read_piece(F[0], 0, 0, i);
    // step t with t % 3 == J: buffer J is multiplied, J + 1 is ready, J + 2 is written from the registers of the same number, which then take
    // a step from memory.  Each product is followed by a share of the other work, in that order: a wavefront issues in order, so work
    // beside a product runs while the matrix core does, and work between groups of products (where the compiler puts it by itself) does not.
    auto step = [&](long long t, auto jc, auto fc) {
      constexpr int J = decltype(jc)::value, J1 = (J + 1) % 3, J2 = (J + 2) % 3, F0 = decltype(fc)::value;
      sum_rows(R[J2], t + 2 < nf);
#pragma unroll
      for (int st = 0; st < NS; ++st) {
        Frags &cur = F[(F0 + st) & 1], &nxt = F[(F0 + st + 1) & 1];
#pragma unroll
        for (int g = 0; g < G; ++g) {
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < NR; ++i)                           // none beside the last quarter: what they bring is needed at once
            if (i * (G - G / 4) / NR == g) read_piece(nxt, st < NS - 1 ? J : J1, st < NS - 1 ? st + 1 : 0, i);
#pragma unroll
          for (int i = 0; i < NQ; ++i)
            if (st == 0 && i * G / NQ == g) stage_piece(R[J2], J2, i);
#pragma unroll
          for (int i = 0; i < NF; ++i)
            if (st == NS - 1 && (NS > 1 ? i * G / NF : G - 1) == g) fetch_piece(R[J2], next, i);
          multiply(cur, g);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      advance();
      __syncthreads();
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    long long t = 0;
    if constexpr (NS % 2 == 0) {
      for (; t + 3 <= nf; t += 3) {
        step(t, I0{}, I0{});
        step(t + 1, I1{}, I0{});
        step(t + 2, I2{}, I0{});
      }
      if (t < nf) step(t, I0{}, I0{});
      if (t + 1 < nf) step(t + 1, I1{}, I0{});
    } else {                                                     // an odd number of fragment sets a step: they change places every step
      for (; t + 6 <= nf; t += 6) {
        step(t, I0{}, I0{});
        step(t + 1, I1{}, I1{});
        step(t + 2, I2{}, I0{});
        step(t + 3, I0{}, I1{});
        step(t + 4, I1{}, I0{});
        step(t + 5, I2{}, I1{});
      }
      if (t < nf) step(t, I0{}, I0{});
      if (t + 1 < nf) step(t + 1, I1{}, I1{});
      if (t + 2 < nf) step(t + 2, I2{}, I0{});
      if (t + 3 < nf) step(t + 3, I0{}, I1{});
      if (t + 4 < nf) step(t + 4, I1{}, I0{});
    }
  }
  if (kt < turns) turn = (int)((kt - nf % turns + turns) % turns);               // the steps of the loop were counted beyond its end
  for (long long m = m0 + nf * BM; m < m1; m += BM) {
    Rows R;
    fetch_masked(R, m);
    sum_rows(R, true);
#pragma unroll
    for (int i = 0; i < NQ; ++i) stage_piece(R, 0, i);
    __syncthreads();
#pragma unroll
    for (int st = 0; st < NS; ++st) {
      Frags F;
#pragma unroll
      for (int i = 0; i < NR; ++i) read_piece(F, 0, st, i);
#pragma unroll
      for (int g = 0; g < G; ++g) multiply(F, g);
    }
    __syncthreads();
  }

  // fp16's last bit is 2^-24 and a code's 2^-9: where all exponents were -15 or more, nothing was lost
  bool wide = false;
  if constexpr (F16) {
    wide = __syncthreads_or(xn > 0 && lowest < -15) != 0;
    if (wide) {                                                  // the chunk's rows again, in bf16: dY's two terms in the first two buffers
#pragma unroll
      for (int a = 0; a < AN; ++a)
#pragma unroll
        for (int b = 0; b < AK; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;
      for (long long m = m0; m < m1; m += BM) {
        Rows R;
        fetch_masked(R, m);
#pragma unroll
        for (int i = 0; i < YP; ++i) {
          u16x8 hi, lo;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = R.y[i].value(e), rest = v - (float)(__bf16)v;
            hi[e] = __builtin_bit_cast(unsigned short, (__bf16)v);
            lo[e] = __builtin_bit_cast(unsigned short, (__bf16)(rest == rest ? rest : 0.f));          // of an infinity or a NaN: none
          }
          *reinterpret_cast<u16x8*>(ly + at<TN>(yr + i * YR, yc)) = hi;
          *reinterpret_cast<u16x8*>(ly + BM * TN + at<TN>(yr + i * YR, yc)) = lo;
        }
#pragma unroll
        for (int j = 0; j < XP; ++j) *reinterpret_cast<u16x8*>(lx + at<TK>(xr, xc + 8 * j)) = widen<false>(R.x[j], pow2f((int)(R.s & 0xffu) - 127));
        __syncthreads();
#pragma unroll
        for (int st = 0; st < NS; ++st) {
          Frags F;
#pragma unroll
          for (int p = 0; p < 2; ++p) {
#pragma unroll
            for (int i = p ? AK : 0; i < NR; ++i) read_piece(F, p, st, i);
#pragma unroll
            for (int g = 0; g < G; ++g) acc[g / AK][g % AK] = mfma<false>(F.a[0][g / AK], F.b[g % AK], acc[g / AK][g % AK]);
          }
        }
        __syncthreads();
      }
    }
  }

  // a lane holds column k = lane & 31 of its blocks; register r is row (r & 3) + 8 (r >> 2) + 4 half
  float* o = out + s * N * K;
#pragma unroll
  for (int b = 0; b < AK; ++b) {
    const int kl = wk * RK + b * 32, k = k0 + kl + (lane & 31);
    const float f = F16 && !wide ? pow2f(top[kl >> 5] - 127 - 7) : 1.f;
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
  if (kt >= turns) return;
  float* sum = reinterpret_cast<float*>(lds);                    // db: the lanes of a column group, in order: [YR][TN]
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[yr * TN + yc + e] = dsum[e];
  __syncthreads();
  for (int c = tid; c < TN; c += NT) {
    float t = 0.f;
    for (int i = 0; i < YR; ++i) t += sum[i * TN + c];
    if (n0 + c < N) dbp[(s * turns + kt) * N + n0 + c] = t;
  }
}

// the largest scale of 32 rows each: tops [ceil(M / 32)][nblk].  A workgroup of the main kernel reads 8 bytes of every row's scales, a cache line
// each: 25 us of 9232 rows.  Here the lines are read whole, once.
__global__ void __launch_bounds__(256)
scale_tops_kernel(const uint8_t* __restrict__ scales, uint8_t* __restrict__ tops, long long M, int nblk, long long n) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const long long g = i / nblk, m = g * 32;
  const uint8_t* p = scales + m * nblk + (i - g * nblk);
  const int rows = M - m < 32 ? (int)(M - m) : 32;
  int t = 0;
  if (rows == 32) {
#pragma unroll
    for (int r = 0; r < 32; ++r) t = max(t, (int)p[(long long)r * nblk]);
  } else {
    for (int r = 0; r < rows; ++r) t = max(t, (int)p[(long long)r * nblk]);
  }
  tops[i] = (uint8_t)t;
}

// dw = gamma sum over the parts + beta db.  Workgroups from `joins` on: db = the sum of the lines of dbp, where dw does not need it
__global__ void __launch_bounds__(256)
wgrad_join_kernel(const float* __restrict__ part, int S, const float* __restrict__ db, const float* __restrict__ gamma, const float* __restrict__ beta,
                  float* __restrict__ dw, long long NK, int K, unsigned joins, const float* __restrict__ dbp, int lines, int N, float* __restrict__ dbo) {
  if (blockIdx.x >= joins) {                                     // 16 columns, 16 lanes each
    __shared__ float buf[16][17];
    const int c = threadIdx.x & 15, l = threadIdx.x >> 4, w = (int)(blockIdx.x - joins) * 16 + c;
    float s = 0.f;
    if (w < N)
#pragma unroll 8
      for (int p = l; p < lines; p += 16) s += dbp[(long long)p * N + w];
    buf[l][c] = s;
    __syncthreads();
    if (l == 0 && w < N) {
#pragma unroll
      for (int i = 1; i < 16; ++i) s += buf[i][c];
      dbo[w] = s;
    }
    return;
  }
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= NK) return;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  const int n = NK - i < 4 ? (int)(NK - i) : 4;
  typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll 4
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

struct WgradShape { int tile, tiles_n, tiles_k, S; long long chunk; int turns; };
// Tile and split by a model of the time (us):
//   a step of 32 rows takes `one` where a CU has one workgroup, and `more` longer for each further one, up to `most` at once; then they go in
//   rounds.  16-bit: tile 256 1.0; 128 0.45 and 0.23; 64 0.43 and 0.22.  f32 (three products): 128 0.98 and 0.58; 64 0.45 and 0.25;
//   S > 1 parts are written and read again at 4.5 TB/s, in a launch of its own.
// The constants were fitted to sweeps over shapes of 100 to 294400 rows and 8 to 4096 columns with an earlier form of the loop (tile 256's step takes
// 0.88 us now).  What they choose is still the fastest of the tiles at each of these, us with tile 256 / 128 / 64, each in its own best split:
//   fp16  36928 x 1024 x 4096 284 / 374 / 1243, 98500 x 768 x 768 134 / 157 / 488, 294400 x 192 x 768 146 / 164 / 374, 73600 x 384 x 1536 125 / 119 / 368,
//         43120 x 512 x 512 63 / 52 / 110, 8192 x 1024 x 1024 47 / 40 / 86, 2000 x 1000 x 1000 34 / 24 / 33, 500 x 2048 x 2048 31 / 17 / 26,
//         100 x 256 x 2048 21 / 10 / 8
//   f32   36928 x 1024 x 4096 - / 900 / 1400, 43120 x 512 x 512 - / 86 / 110, 500 x 2048 x 2048 - / 25 / 27, 100 x 256 x 2048 - / 10 / 7
inline WgradShape wgrad_shape(long long M, int N, int K, int dtype) {
  WgradShape best{};
  double least = 1e300;
  for (int tile : {256, 128, 64}) {
    if (tile == 256 && dtype == OVIS_F32) continue;
    const double one = tile == 256 ? 1.0 : tile == 128 ? (dtype == OVIS_F32 ? 0.98 : 0.45) : (dtype == OVIS_F32 ? 0.45 : 0.43);
    const double more = tile == 256 ? 0.0 : tile == 128 ? (dtype == OVIS_F32 ? 0.58 : 0.23) : (dtype == OVIS_F32 ? 0.25 : 0.22);
    const int most = tile == 256 ? 1 : tile == 128 ? 2 : 4;
    const long long tn = cdiv(N, tile), tk = cdiv(K, tile), tiles = tn * tk;
    long long last = 0;
    for (int want : {1, 128, 256, 512, 1024}) {                  // workgroups in all
      long long S = want / tiles, rows = (M + 63) / 64;
      if (want > 256 * most || want == 1 || S < 1) S = 1;
      if (S > rows) S = rows;
      if (S == last) continue;
      last = S;
      const long long chunk = ((M + S - 1) / S + 31) / 32 * 32, parts = (M + chunk - 1) / chunk, wgs = tiles * parts;
      const long long rounds = (wgs + 256 * most - 1) / (256 * most), per = wgs < 256 * most ? (wgs + 255) / 256 : most;
      const double t = rounds * (chunk / 32) * (one + more * (per - 1)) + (parts > 1 ? 3.0 + 8.0 * parts * N * K / 4.5e6 : 0.0);
      if (t < least) {
        least = t;
        // one part of a few steps: one workgroup sums dY for db, and no second launch adds up what several would have
        best = {tile, (int)tn, (int)tk, (int)parts, chunk, parts == 1 && chunk <= 512 ? 1 : (int)tk};
      }
    }
  }
  return best;
}

// the scales' tops by a launch of their own: where a workgroup's share is 2048 rows or more (below, its own scan is shorter than the launch)
inline bool own_tops(const WgradShape& w, int dtype) { return dtype == OVIS_F16 && w.chunk >= 2048; }
// the workspace: parts of dw and db, the join's sum, tops (4-byte words each)
struct WgradSpace { long long parts, lines, sum, tops; };
inline WgradSpace wgrad_space(const WgradShape& w, long long M, int N, int K, int dtype) {
  const long long NK = (long long)N * K;
  return {w.S * NK, (long long)w.S * w.turns * N, NK < 65536 ? NK : 0, own_tops(w, dtype) ? (M + 31) / 32 * ((K + 31) / 32) / 4 + 1 : 0};
}

}  // namespace

extern "C" long long ovis_linear_wgrad_ckpt8_workspace_bytes(long long M, int N, int K, int dtype) {
  if (M <= 0 || N <= 0 || K <= 0 || !ovis::dtype_ok(dtype)) return 0;
  const WgradShape w = wgrad_shape(M, N, K, dtype);
  const WgradSpace p = wgrad_space(w, M, N, K, dtype);
  return (p.parts + p.lines + p.sum + p.tops) * 4;
}

extern "C" int ovis_linear_wgrad_ckpt8(const void* dy, long long lddy, const uint8_t* codes, const uint8_t* scales, const float* gamma,
                                       const float* beta, float* dw, float* db, float* workspace, long long M, int N, int K, int dtype,
                                       ovis_stream_t stream) {
  OVIS_REQUIRE(dy && codes && scales && dw && db && workspace && (!gamma == !beta), "linear_wgrad_ckpt8: null pointer");
  OVIS_REQUIRE(M > 0 && N > 0 && K > 0 && lddy >= N && ovis::dtype_ok(dtype), "linear_wgrad_ckpt8: M %lld, N %d, K %d, row stride %lld, type %d", M, N,
               K, lddy, dtype);
  const WgradShape w = wgrad_shape(M, N, K, dtype);
  const long long blocks = (long long)w.tiles_n * w.tiles_k * w.S;
  OVIS_REQUIRE(blocks <= ovis::kMostBlocks && (long long)N * K < (1ll << 33) && lddy < (1ll << 24) && K < (1 << 24), "linear_wgrad_ckpt8: %d x %d (row stride %lld) is too large for one call", N,
               K, lddy);
  const bool join = w.S > 1 || gamma;
  float* part = join ? workspace : dw;
  const int lines = w.S * w.turns;
  const WgradSpace sp = wgrad_space(w, M, N, K, dtype);
  float* dbp = lines > 1 ? workspace + sp.parts : db;
  const uint8_t* tops = scales;
  int tshift = 0;
  if (own_tops(w, dtype)) {
    uint8_t* t = (uint8_t*)(workspace + sp.parts + sp.lines + sp.sum);
    const long long n = (M + 31) / 32 * ((K + 31) / 32);
    hipLaunchKernelGGL(scale_tops_kernel, dim3(ovis::cdiv(n, 256)), dim3(256), 0, (hipStream_t)stream, scales, t, M, (K + 31) / 32, n);
    const int rc = ovis::check_launch("linear_wgrad_ckpt8");
    if (rc != OVIS_OK) return rc;
    tops = t, tshift = 5;
  }
#define WG_GO(T, TN, TK, WN, WK, BM)                                                                                                        \
  {                                                                                                                                         \
    const int lds = 3 * BM * (TN * (sizeof(T) == 4 ? 3 : 1) + TK) * 2;                                                                      \
    if (lds > 65536) {                                                                                                                      \
      const hipError_t e = hipFuncSetAttribute((const void*)wgrad_ckpt8_kernel<T, TN, TK, WN, WK, BM>,                                      \
                                               hipFuncAttributeMaxDynamicSharedMemorySize, lds);                                            \
      if (e != hipSuccess) return ovis::fail(OVIS_ELAUNCH, "linear_wgrad_ckpt8: %s", hipGetErrorString(e));                                 \
    }                                                                                                                                       \
    hipLaunchKernelGGL((wgrad_ckpt8_kernel<T, TN, TK, WN, WK, BM>), dim3((unsigned)blocks), dim3(64 * WN * WK), lds, (hipStream_t)stream,   \
                       (const T*)dy, lddy, codes, scales, part, dbp, M, N, K, w.chunk, w.tiles_n, w.tiles_k, w.turns, tops, tshift);        \
  }
  if (dtype == OVIS_F32) {
    if (w.tile == 128) WG_GO(float, 128, 128, 2, 2, 16)
    else WG_GO(float, 64, 64, 2, 2, 32)
  } else if (dtype == OVIS_F16) {
    if (w.tile == 256) WG_GO(_Float16, 256, 256, 2, 2, 32)
    else if (w.tile == 128) WG_GO(_Float16, 128, 128, 2, 2, 32)
    else WG_GO(_Float16, 64, 64, 2, 2, 32)
  } else {
    if (w.tile == 256) WG_GO(__bf16, 256, 256, 2, 2, 32)
    else if (w.tile == 128) WG_GO(__bf16, 128, 128, 2, 2, 32)
    else WG_GO(__bf16, 64, 64, 2, 2, 32)
  }
#undef WG_GO
  int rc = ovis::check_launch("linear_wgrad_ckpt8");
  if (rc != OVIS_OK) return rc;
  const long long NK = (long long)N * K;
  int S = w.S;
  const bool tree = S > 8 && NK < 65536, later = join && !tree && !gamma;         // db's lines are added up beside dw's parts where that can be
  if (lines > 1 && !tree && !later) rc = ovis::column_sum_finish(dbp, lines, N, db, N, db, (hipStream_t)stream);
  if (rc != OVIS_OK || !join) return rc;
  if (tree) {                                     // few columns, many parts: 64 lanes a column (9000 x 64 x 64 in 141 parts: 57 us by one)
    float* to = gamma ? workspace + sp.parts + sp.lines : dw;
    rc = ovis::column_sum_two({part, S, (int)NK, to, (int)NK, to}, {dbp, lines, N, db, N, db}, (hipStream_t)stream);
    if (rc != OVIS_OK || !gamma) return rc;
    part = to;
    S = 1;
  }
  const unsigned joins = ovis::cdiv((NK + 3) / 4, 256);
  hipLaunchKernelGGL(wgrad_join_kernel, dim3(joins + (later && lines > 1 ? ovis::cdiv(N, 16) : 0)), dim3(256), 0, (hipStream_t)stream, part, S,
                     gamma ? db : nullptr, gamma, beta, dw, NK, K, joins, dbp, lines, N, db);
  return ovis::check_launch("linear_wgrad_ckpt8");
}
