// Layer norm for training on gfx950: forward with the row statistics and, if asked, the normalised rows in 8 bits; backward with the input,
// weight and bias gradients.
//
//   s    = x + residual, rounded to x's type (what the next layer and the backward pass see)
//   xhat = (s - mean) * rstd,  y = xhat * gamma + beta           mean, rstd = 1/sqrt(var + eps): two passes over registers, f32
//   gd   = dy * gamma
//   dx   = rstd * (gd - mean(gd) - xhat * mean(gd * xhat)) + dsum
//   dgamma = sum over rows dy * xhat,  dbeta = sum over rows dy
//
// Bound by HBM: every input is read once and every output written once.  LPR neighbouring lanes hold a row in registers, 8 columns a lane and
// NCH such pieces each (up to 256 lanes, a whole workgroup), so a row is read once although forward needs it three times.
// The weight gradient is summed over rows in a fixed order: a workgroup keeps the sums of its rows in registers, writes one line of the
// workspace, and a second kernel adds the lines (no atomics: the same bits at every call).
#include "train_elem.h"

namespace {

using namespace ovis;

// sums over the LPR lanes of a row, N of them side by side: moves between lanes of the vector unit, no LDS (by LDS permutes a step takes ten times
// as long, and a row's sums are a chain of them).  LPR = 256 crosses the four wavefronts through `buf`, with one barrier: the caller alternates
// between two of them.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int LPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (&buf)[N][4]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float t = v[i];
    t = dpp_add<0xB1>(t);                                        // lanes 1 0 3 2 of four
    t = dpp_add<0x4E>(t);                                        // lanes 2 3 0 1
    t = dpp_add<0x141>(t);                                       // mirrored within eight: the other four
    t = dpp_add<0x140>(t);                                       // mirrored within sixteen: the other eight
    if constexpr (LPR >= 32) {
      const unsigned u = __builtin_bit_cast(unsigned, t);
      const auto w = __builtin_amdgcn_permlane16_swap(u, u, false, false);         // the even and the odd sixteens
      t = __builtin_bit_cast(float, (unsigned)w[0]) + __builtin_bit_cast(float, (unsigned)w[1]);
    }
    if constexpr (LPR >= 64) {
      const unsigned u = __builtin_bit_cast(unsigned, t);
      const auto w = __builtin_amdgcn_permlane32_swap(u, u, false, false);
      t = __builtin_bit_cast(float, (unsigned)w[0]) + __builtin_bit_cast(float, (unsigned)w[1]);
    }
    v[i] = t;
  }
  if constexpr (LPR > 64) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((threadIdx.x & 63) == 0) buf[i][threadIdx.x >> 6] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (LPR == 128) v[i] = threadIdx.x < 128 ? buf[i][0] + buf[i][1] : buf[i][2] + buf[i][3];
      else v[i] = (buf[i][0] + buf[i][1]) + (buf[i][2] + buf[i][3]);
    }
  }
}

template <typename TX, typename TY, int LPR, int NCH>
__global__ void __launch_bounds__(256)
layernorm_train_fwd_kernel(const TX* __restrict__ x, long long ldx, const TX* __restrict__ res, long long ldr, const float* __restrict__ gamma,
                           const float* __restrict__ beta, TX* __restrict__ sum, TY* __restrict__ y, float* __restrict__ stats,
                           uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, long long rows, int C, float eps) {
  __shared__ float buf[2][1][4];
  const int li = threadIdx.x % LPR;
  const long long row = (long long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const bool live = row < rows;                                  // lanes of a row behind the last one stay for the shuffles
  const long long r = live ? row : rows - 1;
  const bool on = row + 8 < rows;                                // eight rows on, a row's end is not the tensor's
  float v[NCH][8];
  float s[1] = {0.f}, q[1] = {0.f};
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = (c * LPR + li) * 8, n = C - col;
    if (n > 0) {
      load8(x + r * ldx + col, n, on, v[c]);
      if (res) {
        float t[8];
        load8(res + r * ldr + col, n, on, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] = (float)(TX)(v[c][e] + t[e]);
        if (live) store8(sum + r * C + col, n, v[c]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s[0] += v[c][e];
  }
  row_sums<LPR>(s, buf[0]);
  const float mean = s[0] / (float)C;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int n = C - (c * LPR + li) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[c][e] = e < n ? v[c][e] - mean : 0.f;
      q[0] += v[c][e] * v[c][e];
    }
  }
  row_sums<LPR>(q, buf[1]);
  const float rstd = 1.f / sqrtf(q[0] / (float)C + eps);
  if (live && li == 0) {
    stats[2 * r] = mean;
    stats[2 * r + 1] = rstd;
  }
  const int nblk = (C + 31) >> 5;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = (c * LPR + li) * 8, n = C - col;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[c][e] *= rstd;
    if (codes) {                                                 // all four lanes of a block take part, the ones behind the row's end with 0
      unsigned sb;
      const u32x2_u q8 = encode8(v[c], false, sb);
      if (live && n > 0) {
        store_codes(codes + r * C + col, n, q8);
        if ((li & 3) == 0) scales[r * nblk + (col >> 5)] = (uint8_t)sb;
      }
    }
    if (live && n > 0) {
      float g[8], b[8];
      load8(gamma + col, n, g);
      load8(beta + col, n, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = v[c][e] * g[e] + b[e];
      store8(y + r * C + col, n, v[c]);
    }
  }
}

// TX: x, dsum and dx; TY: dy; CK: the normalised rows come in 8 bits; TAIL: C is no multiple of 8, a row's last piece is masked (a variant of its
// own: a mask in the other costs it the fetch ahead, 109 -> 144 us).  A workgroup walks over rows and keeps dgamma / dbeta of its lanes' columns
// in registers, gamma in LDS.  The next row is fetched before the present one's sums begin, and rows stay in their stored width until they are
// used: the sums take two dependent passes over a row, in which a wavefront without the next row's loads would have nothing in flight.
// 98500 x 768 fp16 from 8 bits with dsum: 108 us, 4.9 TB/s (without the fetch ahead 133 us; a large copy reaches 5.0 TB/s).
template <typename TX, typename TY, bool CK, bool TAIL, int LPR, int NCH, int WAVES>
__global__ void __launch_bounds__(256, WAVES)
layernorm_train_bwd_kernel(const TY* __restrict__ dy, long long lddy, const TX* __restrict__ x, long long ldx, const uint8_t* __restrict__ codes,
                           const uint8_t* __restrict__ scales, const float* __restrict__ stats, const float* __restrict__ gamma,
                           const TX* __restrict__ dsum, long long ldds, TX* __restrict__ dx, float* __restrict__ part, long long rows, int C) {
  __shared__ float buf[2][2][4];
  extern __shared__ float acc[];                                 // [2][Cp]: gamma in the first line, at the end the workgroup's sums
  const int li = threadIdx.x % LPR, Cp = NCH * LPR * 8;
  constexpr int RPB = 256 / LPR;
  const int nblk = (C + 31) >> 5;
  for (int i = threadIdx.x; i < Cp; i += 256) acc[i] = i < C ? gamma[i] : 0.f;
  __syncthreads();
  float dg[NCH][8], db[NCH][8];
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) dg[c][e] = db[c][e] = 0.f;
  Raw8<TY> dn[NCH];                                              // the next row's
  Raw8<TX> hn[NCH], tn[NCH];
  u32x2_u qn[NCH];
  unsigned qsn[NCH];
  float meann, rstdn;
  auto fetch = [&](long long row) {
    const bool live = row < rows, on = row + 8 < rows;           // eight rows on, a row's end is not the tensor's
    const long long r = live ? row : rows - 1;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * LPR + li) * 8, n = live ? C - col : 0;
      if constexpr (TAIL) dn[c].load(dy + r * lddy + col, n, on);
      else dn[c].load_all(dy + r * lddy + col, n > 0);
      if constexpr (CK) {
        qn[c] = TAIL ? load_codes(codes + r * C + col, n, on) : load_codes(codes + r * C + col, n > 0 ? 8 : 0);
        qsn[c] = n > 0 ? scales[r * nblk + (col >> 5)] : 127u;
      } else {
        if constexpr (TAIL) hn[c].load(x + r * ldx + col, n, on);
        else hn[c].load_all(x + r * ldx + col, n > 0);
      }
    }
    meann = stats[2 * r], rstdn = stats[2 * r + 1];
    if (dsum)
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int col = (c * LPR + li) * 8;
        if constexpr (TAIL) tn[c].load(dsum + r * ldds + col, live ? C - col : 0, on);
        else tn[c].load_all(dsum + r * ldds + col, live && C > col);
      }
  };
  int phase = 0;
  fetch((long long)blockIdx.x * RPB + threadIdx.x / LPR);
  for (long long r0 = (long long)blockIdx.x * RPB; r0 < rows; r0 += (long long)gridDim.x * RPB) {
    const long long row = r0 + threadIdx.x / LPR;
    const bool live = row < rows;
    const long long r = live ? row : rows - 1;
    Raw8<TY> d[NCH];
    Raw8<TX> h[NCH], t[NCH];
    u32x2_u q[NCH];
    unsigned qs[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) d[c] = dn[c], h[c] = hn[c], t[c] = tn[c], q[c] = qn[c], qs[c] = qsn[c];
    const float mean = meann, rstd = rstdn;
    if (r0 + (long long)gridDim.x * RPB < rows) fetch(row + (long long)gridDim.x * RPB);
    auto xhat = [&](int c, float (&v)[8]) {
      if constexpr (CK) {
        decode8(q[c], qs[c], v);
      } else {
        const int n = live ? C - (c * LPR + li) * 8 : 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? (h[c].at(e) - mean) * rstd : 0.f;
      }
    };
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const float* g = acc + (c * LPR + li) * 8;
      const int n = C - (c * LPR + li) * 8;
      float v[8];
      xhat(c, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (TAIL && CK) v[e] = e < n ? v[e] : 0.f;     // without codes xhat has done so
        const float de = TAIL && e >= n ? 0.f : d[c].at(e), gd = de * g[e];
        s[0] += gd;
        s[1] += gd * v[e];
        dg[c][e] += de * v[e];
        db[c][e] += de;
      }
    }
    row_sums<LPR>(s, buf[phase]);
    const float c1 = s[0] / (float)C, c2 = s[1] / (float)C;
    phase ^= 1;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {                              // from here on the stored forms are widened again, not kept widened
      d[c].hide();
      if constexpr (CK) hide(q[c]);
      else h[c].hide();
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * LPR + li) * 8, n = live ? C - col : 0;
      const float* g = acc + col;
      float v[8], o[8];
      xhat(c, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = rstd * (d[c].at(e) * g[e] - c1 - v[e] * c2);
      if (dsum)
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] += t[c].at(e);
      if (n > 0) store8(dx + r * C + col, n, o);
    }
  }
  // the rows of a workgroup, in order: lanes of the same columns are LPR apart
  __syncthreads();
  for (int k = 0; k < RPB; ++k) {
    if ((int)threadIdx.x / LPR == k) {
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int col = (c * LPR + li) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          acc[col + e] = (k ? acc[col + e] : 0.f) + dg[c][e];
          acc[Cp + col + e] = (k ? acc[Cp + col + e] : 0.f) + db[c][e];
        }
      }
    }
    __syncthreads();
  }
  float* line = part + (long long)blockIdx.x * 2 * C;
  for (int i = threadIdx.x; i < C; i += 256) {
    line[i] = acc[i];
    line[C + i] = acc[Cp + i];
  }
}

struct RowShape { int lpr, nch; };
// Lanes per row: the fewest that hold the row in `most` pieces each, since a lane's extra pieces are loads in flight while a lane behind the
// row's end is idle.  128 lanes in two pieces are no gain over 256 in one for 16-bit rows (27286 x 1800 backward 83 us against 78; 27286 x 3000 in
// three pieces 119 us, by 256 lanes in two 179 us; f32 of 1600 columns 62 us against 70).
inline RowShape row_shape(int C, int most) {
  const int nvec = (C + 7) / 8;
  for (int lpr : {16, 32, 64, 128, 256}) {
    const int nch = (nvec + lpr - 1) / lpr;
    if (nch <= most && !(most == 3 && lpr == 128 && nch < 3)) return {lpr, nch};
  }
  return {256, (nvec + 255) / 256};                              // C <= 8192: at most four
}
// Backward: a piece is 16 sums and two rows' dy, x and dsum: three pieces of 16-bit rows (220 registers) or two of f32 rows (192), two
// wavefronts a SIMD; two pieces of 16-bit rows (165), three wavefronts (27286 x 4096: 147 us, with two wavefronts 169 us).  Before the fetch ahead
// 98500 x 768 fp16 took 133 us in three pieces, 144 us in two; 73600 x 384 f32 87 us in three, 83 us in two.  Rows of more than 4096 f32 or 6144
// 16-bit columns need more registers and spill.
inline RowShape bwd_row_shape(int C, int x_dtype) { return row_shape(C, x_dtype == OVIS_F32 ? 2 : 3); }

// as many workgroups as the card holds at once: each walks over its rows, and a workgroup that had to wait would walk alone at the end
constexpr int bwd_waves(int nch, bool f32) { return nch == 1 ? 4 : nch == 2 && !f32 ? 3 : 2; }
inline unsigned bwd_blocks(long long rows, const RowShape& s, int x_dtype) {
  const long long need = (rows + 256 / s.lpr - 1) / (256 / s.lpr), full = 256 * bwd_waves(s.nch, x_dtype == OVIS_F32);
  if (need <= 4) return 1;                                       // and no second launch: the workgroup's sums are the gradients
  const long long most = rows / 10 < 256 ? 256 : rows / 10 < full ? rows / 10 : full;    // a workgroup's line of sums costs as much as three rows
  return (unsigned)(need < most ? need : most);
}

}  // namespace

namespace ovis {

// out0[w] (w < split), out1[w - split] = sum over the P lines of part [P][W], in a fixed order.  Two forms:
// narrow: 64 lanes of a column take every 64th line, then a tree; 16 columns a workgroup, so that the lines, which come from L2, are read by
// many workgroups.  wide: a lane takes four columns and all lines.  The wide form needs no exchange but fills the card only from
// tens of thousands of columns on: 33 lines of 124416 columns 5 us against 20, 126 lines of 29282 columns 40 us against 6.
__global__ void __launch_bounds__(1024)
column_sum_narrow_kernel(ColumnSum a, ColumnSum b, unsigned first) {             // workgroups from `first` on: b
  __shared__ float buf[64][17];
  const ColumnSum& k = blockIdx.x < first ? a : b;
  const float* part = k.part;
  const int P = k.P, W = k.W;
  const int c = threadIdx.x & 15, p0 = threadIdx.x >> 4;
  const int w = (blockIdx.x - (blockIdx.x < first ? 0 : first)) * 16 + c;
  float s = 0.f;
  if (w < W)
    for (int p = p0; p < P; p += 64) s += part[(long long)p * W + w];
  buf[p0][c] = s;
  __syncthreads();
  for (int o = 32; o > 0; o >>= 1) {
    if (p0 < o) buf[p0][c] += buf[p0 + o][c];
    __syncthreads();
  }
  if (p0 == 0 && w < W) {
    if (w < k.split) k.out0[w] = buf[0][c];
    else k.out1[w - k.split] = buf[0][c];
  }
}

__global__ void __launch_bounds__(256)
column_sum_wide_kernel(const float* __restrict__ part, int P, int W, float* __restrict__ out0, int split, float* __restrict__ out1) {
  const long long w = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (w >= W) return;
  typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
  f32x4_u s = {0.f, 0.f, 0.f, 0.f};
  const int n = W - w < 4 ? (int)(W - w) : 4;
  if (n == 4) {
#pragma unroll 8
    for (int p = 0; p < P; ++p) {
      const f32x4_u t = *reinterpret_cast<const f32x4_u*>(part + (long long)p * W + w);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += t[e];
    }
  } else {
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (e < n) s[e] += part[(long long)p * W + w + e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (e < n) {
      if (w + e < split) out0[w + e] = s[e];
      else out1[w + e - split] = s[e];
    }
  }
}

int column_sum_finish(const float* part, int P, int W, float* out0, int split, float* out1, hipStream_t stream) {
  if (W >= 65536)
    hipLaunchKernelGGL(column_sum_wide_kernel, dim3(cdiv(W, 1024)), dim3(256), 0, stream, part, P, W, out0, split, out1);
  else
    hipLaunchKernelGGL(column_sum_narrow_kernel, dim3(cdiv(W, 16)), dim3(1024), 0, stream, ColumnSum{part, P, W, out0, split, out1}, ColumnSum{}, cdiv(W, 16));
  return check_launch("column_sum_finish");
}

int column_sum_two(const ColumnSum& a, const ColumnSum& b, hipStream_t stream) {
  const unsigned first = cdiv(a.W, 16);
  hipLaunchKernelGGL(column_sum_narrow_kernel, dim3(first + cdiv(b.W, 16)), dim3(1024), 0, stream, a, b, first);
  return check_launch("column_sum_two");
}

}  // namespace ovis

#define LN_TYPES(xt, yt, WIDE, NARROW)                                                              \
  if (xt == OVIS_F32 && yt == OVIS_F32) { LN_SWITCH(WIDE(float, float)) }                           \
  else if (xt == OVIS_F32 && yt == OVIS_F16) { LN_SWITCH(WIDE(float, _Float16)) }                   \
  else if (xt == OVIS_F32) { LN_SWITCH(WIDE(float, __bf16)) }                                       \
  else if (xt == OVIS_F16) { LN_SWITCH(NARROW(_Float16, _Float16)) }                                \
  else { LN_SWITCH(NARROW(__bf16, __bf16)) }
#define LN_SWITCH(cases)                                                                            \
  switch (sh.lpr * 8 + sh.nch) {                                                                    \
    cases                                                                                           \
    default: return ovis::fail(OVIS_EINVAL, "layernorm_train: no kernel for rows of %d", C);        \
  }
#define LN_CASE(TX, TY, LPR, NCH) case LPR * 8 + NCH: LN_GO(TX, TY, LPR, NCH); break;
// the shapes that row_shape(C, 4), (C, 3) and (C, 2) give
#define LN_MOST4(TX, TY)                                                                            \
  LN_CASE(TX, TY, 16, 1) LN_CASE(TX, TY, 16, 2) LN_CASE(TX, TY, 16, 3) LN_CASE(TX, TY, 16, 4)       \
  LN_CASE(TX, TY, 32, 3) LN_CASE(TX, TY, 32, 4) LN_CASE(TX, TY, 64, 3) LN_CASE(TX, TY, 64, 4) LN_CASE(TX, TY, 128, 3)             \
  LN_CASE(TX, TY, 128, 4) LN_CASE(TX, TY, 256, 3) LN_CASE(TX, TY, 256, 4)
#define LN_MOST3(TX, TY)                                                                            \
  LN_CASE(TX, TY, 16, 1) LN_CASE(TX, TY, 16, 2) LN_CASE(TX, TY, 16, 3) LN_CASE(TX, TY, 32, 2)       \
  LN_CASE(TX, TY, 32, 3) LN_CASE(TX, TY, 64, 2) LN_CASE(TX, TY, 64, 3) LN_CASE(TX, TY, 128, 3) LN_CASE(TX, TY, 256, 1)             \
  LN_CASE(TX, TY, 256, 2) LN_CASE(TX, TY, 256, 3) LN_CASE(TX, TY, 256, 4)
#define LN_MOST2(TX, TY)                                                                            \
  LN_CASE(TX, TY, 16, 1) LN_CASE(TX, TY, 16, 2) LN_CASE(TX, TY, 32, 2) LN_CASE(TX, TY, 64, 2)       \
  LN_CASE(TX, TY, 128, 2) LN_CASE(TX, TY, 256, 2) LN_CASE(TX, TY, 256, 3) LN_CASE(TX, TY, 256, 4)

extern "C" int ovis_layernorm_train_forward(const void* x, long long ldx, const void* residual, long long ldr, const float* gamma,
                                            const float* beta, void* sum, void* y, float* stats, uint8_t* codes, uint8_t* scales,
                                            long long rows, int C, float eps, int x_dtype, int y_dtype, ovis_stream_t stream) {
  OVIS_REQUIRE(x && gamma && beta && y && stats && (!residual || sum) && (!codes == !scales), "layernorm_train_forward: null pointer");
  OVIS_REQUIRE(rows > 0 && C > 0 && C <= 8192, "layernorm_train_forward: rows %lld, columns %d (1 to 8192)", rows, C);
  OVIS_REQUIRE(ldx >= C && (!residual || ldr >= C), "layernorm_train_forward: row stride below the row length");
  OVIS_REQUIRE(ovis::dtype_ok(x_dtype) && ovis::dtype_ok(y_dtype) && (x_dtype == OVIS_F32 || x_dtype == y_dtype),
               "layernorm_train_forward: y has x's type, or any where x is f32");
  const RowShape sh = row_shape(C, 4);
  const long long blocks = (rows + 256 / sh.lpr - 1) / (256 / sh.lpr);
  OVIS_REQUIRE(blocks <= ovis::kMostBlocks, "layernorm_train_forward: %lld rows are too many for one launch", rows);
#define LN_GO(TX, TY, LPR, NCH)                                                                                                             \
  hipLaunchKernelGGL((layernorm_train_fwd_kernel<TX, TY, LPR, NCH>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream,            \
                     (const TX*)x, ldx, (const TX*)residual, ldr, gamma, beta, (TX*)sum, (TY*)y, stats, codes, scales, rows, C, eps)
  LN_TYPES(x_dtype, y_dtype, LN_MOST4, LN_MOST4)
#undef LN_GO
  return ovis::check_launch("layernorm_train_forward");
}

extern "C" long long ovis_layernorm_train_backward_workspace_bytes(long long rows, int C, int x_dtype) {
  if (rows <= 0 || C <= 0 || C > 8192 || !ovis::dtype_ok(x_dtype)) return 0;
  return (long long)bwd_blocks(rows, bwd_row_shape(C, x_dtype), x_dtype) * 2 * C * 4;
}

extern "C" int ovis_layernorm_train_backward(const void* dy, long long lddy, const void* x, long long ldx, const uint8_t* codes,
                                             const uint8_t* scales, const float* stats, const float* gamma, const void* dsum, long long ldds,
                                             void* dx, float* dgamma, float* dbeta, float* workspace, long long rows, int C, int dy_dtype,
                                             int x_dtype, ovis_stream_t stream) {
  OVIS_REQUIRE(dy && stats && gamma && dx && dgamma && dbeta && workspace && (!codes == !scales) && (!x != !codes),
               "layernorm_train_backward: null pointer, or not exactly one of x and codes");
  OVIS_REQUIRE(rows > 0 && C > 0 && C <= 8192, "layernorm_train_backward: rows %lld, columns %d (1 to 8192)", rows, C);
  OVIS_REQUIRE(lddy >= C && (!x || ldx >= C) && (!dsum || ldds >= C), "layernorm_train_backward: row stride below the row length");
  OVIS_REQUIRE(ovis::dtype_ok(dy_dtype) && ovis::dtype_ok(x_dtype) && (x_dtype == OVIS_F32 || x_dtype == dy_dtype),
               "layernorm_train_backward: dy has x's type, or any where x is f32");
  const RowShape sh = bwd_row_shape(C, x_dtype);
  const unsigned blocks = bwd_blocks(rows, sh, x_dtype);
  float* to = blocks == 1 && dbeta == dgamma + C ? dgamma : workspace;
#define LN_GO(TX, TY, LPR, NCH)                                                                                                             \
  if (codes && C % 8) LN_RUN(TX, TY, true, true, LPR, NCH);                                                                                 \
  else if (codes) LN_RUN(TX, TY, true, false, LPR, NCH);                                                                                    \
  else if (C % 8) LN_RUN(TX, TY, false, true, LPR, NCH);                                                                                    \
  else LN_RUN(TX, TY, false, false, LPR, NCH)
#define LN_RUN(TX, TY, CK, TAIL, LPR, NCH)                                                                                                  \
  hipLaunchKernelGGL((layernorm_train_bwd_kernel<TX, TY, CK, TAIL, LPR, NCH, bwd_waves(NCH, sizeof(TX) == 4)>), dim3(blocks),                                \
                     dim3(256), 2 * LPR * NCH * 8 * 4, (hipStream_t)stream, (const TY*)dy, lddy, (const TX*)x, ldx, codes, scales, stats,   \
                     gamma, (const TX*)dsum, ldds, (TX*)dx, to, rows, C)
  LN_TYPES(x_dtype, dy_dtype, LN_MOST2, LN_MOST3)
#undef LN_GO
#undef LN_RUN
  const int rc = ovis::check_launch("layernorm_train_backward");
  if (rc != OVIS_OK || to != workspace) return rc;
  return ovis::column_sum_finish(workspace, (int)blocks, 2 * C, dgamma, C, dbeta, (hipStream_t)stream);
}
