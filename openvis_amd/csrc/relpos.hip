// Learned relative position bias by buckets, and the gradient of its table (gfx950).
//
//   sequences   bias[h, i, j] = table[bucket(j - i - q_offset), h]: the bucket of a distance is monotone in it on either side of 0, so a bucket
//               is one run of diagonals and the host hands over the runs' borders (distances at which the next bucket begins)
//   windows     bias[h, i, j] = table[(yi - yj + ws - 1)(2 ws - 1) + xi - xj + ws - 1, h] (forward: swin_ops.hip)
//   gradient    dtable[b, h] = sum over the batch and all (i, j) of bucket b of dbias[., h, i, j]
//
// Bound by HBM: forward writes the bias once, backward reads the gradient once.  All sums are taken in a fixed order.
#include "train_elem.h"

namespace {

using namespace ovis;

constexpr int kMaxBuckets = 256;
// borders of the buckets of one direction, ascending: bucket = number of borders <= distance; by value, as a kernel argument
struct Borders { int n; int at[kMaxBuckets]; };

__device__ __forceinline__ int bucket_of(long long r, const int* at, int n, int both) {
  const long long d = both ? (r < 0 ? -r : r) : (r < 0 ? -r : 0);
  int lo = 0, hi = n;                                            // at[0] >= 1: bucket 0 is distance 0
  while (lo < hi) {
    const int m = (lo + hi) >> 1;
    if (d >= at[m]) lo = m + 1;
    else hi = m;
  }
  return lo + (both && r > 0 ? n + 1 : 0);
}

// the bucket's r = j - i - off, as a run [r0, r1)
__device__ __forceinline__ void bucket_run(int bk, const int* at, int n, int both, long long& r0, long long& r1) {
  const int side = n + 1;
  const bool pos = both && bk >= side;
  const int k = pos ? bk - side : bk;
  const long long far = 1ll << 61, first = k == 0 ? 0 : at[k - 1], last = k == n ? far : at[k];      // magnitudes [first, last)
  r0 = pos ? (first > 1 ? first : 1) : 1 - last;
  r1 = pos ? last : k == 0 && !both ? far : 1 - first;                                                     // one direction: r > 0 is distance 0 too
}

// A workgroup writes 256 V columns (V = 16 bytes) of a run of rows of one head.  Row i + 1 is row i moved one column on, so the values of all
// its diagonals are laid out once in LDS and a lane holds its V columns in registers, takes one new value a row and moves the others on.
template <typename T>
__global__ void __launch_bounds__(256)
relpos_fwd_kernel(const float* __restrict__ table, T* __restrict__ out, Borders b, int both, int H, int Nq, int Nk, int ld, long long off,
                  int rows) {
  constexpr int V = 16 / sizeof(T);
  extern __shared__ unsigned char raw[];
  T* line = reinterpret_cast<T*>(raw);                           // line[k]: diagonal j - i = c0 - (i1 - 1) + k
  const int h = blockIdx.z, i0 = blockIdx.y * rows, i1 = min(i0 + rows, Nq), c0 = blockIdx.x * 256 * V;
  const int len = min(256 * V, ld - c0) + (i1 - i0) - 1;
  __shared__ int at[kMaxBuckets];                                // the borders and the head's values: a search in LDS takes a fraction of one
  __shared__ float val[2 * (kMaxBuckets + 1)];                   // through the arguments' memory
  for (int k = threadIdx.x; k < b.n; k += 256) at[k] = b.at[k];
  for (int k = threadIdx.x; k < (b.n + 1) * (both ? 2 : 1); k += 256) val[k] = table[(long long)k * H + h];
  __syncthreads();
  for (int k = threadIdx.x; k < len; k += 256) line[k] = (T)val[bucket_of((long long)c0 - (i1 - 1) + k - off, at, b.n, both)];
  __syncthreads();
  const int c = c0 + threadIdx.x * V;
  if (c >= ld) return;                                           // ld % V == 0
  typedef T vec __attribute__((ext_vector_type(V)));
  vec v;
  const T* p = line + threadIdx.x * V + (i1 - 1 - i0);           // p[e]: column c + e of row i0
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = p[e];
  T* o = out + ((long long)h * Nq + i0) * ld + c;
  for (int i = i0; i < i1; ++i) {
    vec w = v;
    if (c + V > Nk) {
#pragma unroll
      for (int e = 0; e < V; ++e) w[e] = c + e < Nk ? v[e] : (T)0.f;
    }
    *reinterpret_cast<vec*>(o) = w;
    o += ld;
#pragma unroll
    for (int e = V - 1; e > 0; --e) v[e] = v[e - 1];
    if (i + 1 < i1) v[0] = *--p;
  }
}

// Times below are of calls on one input again and again; the 134 MB of 8 x 8 x 1023^2 bf16 then stay in the last-level cache, where a call takes 35 us.
// From memory, on inputs that take turns, it takes 46 us.
//
// Rows of a lane that are fetched at once: eight (8 x 8 x 1023^2 bf16 37 us, by fours 40 us); four where rows are so short that most of eight
// would lie outside (9 x 20 x 3834 x 32 f32 34 us, by eights 42 us).
constexpr int rows_in_flight(int lanes) { return lanes == 8 ? 4 : 8; }

// Diagonal sums.  A wavefront owns 64 V diagonals, V neighbouring ones a lane, and walks down the rows of its share: the lane's V elements
// of the next row lie one element on, so they are loaded as one vector at any element's address and added to the same registers -- no
// transposition, no LDS, no atomics.  Where a row is short, L < 64 lanes take 8 L diagonals and 64 / L rows go at once: a strip of 8 L diagonals
// meets rows of Nk columns, so 8 L beyond Nk is idle (9 x 20 x 3834 x 32 f32: 102 us with 64 lanes).  A vector that crosses an end of its row is read all the
// same, from the neighbouring rows' elements, and masked; only where it would leave the tensor's span (first and last rows) are its elements read one by one: a separate read of a row's ends
// cost more than the rows themselves (8 x 8 x 1023^2 bf16: 50 us).  A workgroup is four wavefronts on the same diagonals, rows dealt in turn;
// it adds its diagonals up by buckets, 16 lanes a bucket, into one line of the workspace [buckets][H] (a line of diagonals and a launch that
// sums them afterwards: 4 to 5 us more).  grid: (diagonal strips, row chunks x batch, heads).
template <typename T, int L>
__global__ void __launch_bounds__(256)
relpos_bwd_kernel(const T* __restrict__ g, long long bs, long long hs, long long ld, float* __restrict__ part, Borders borders, int both,
                  long long off, long long B, long long bper, int Nq, int Nk, int rows, int chunks) {
  constexpr int V = 8, U = rows_in_flight(L), RG = 256 / L;      // RG row groups
  __shared__ float buf[RG][L * V + 4];
  __shared__ int edge[kMaxBuckets];                              // the borders: searched at the end, read from the arguments' memory (slow) at once
  const int mine = (int)threadIdx.x < borders.n ? borders.at[threadIdx.x] : 0;
  const int lane = threadIdx.x % L;
  const int grp = L == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : threadIdx.x / L;
  const int h = blockIdx.z, ck = blockIdx.y % chunks;
  const long long b0 = (long long)(blockIdx.y / chunks) * bper, b1 = b0 + bper < B ? b0 + bper : B;
  const long long span = (B - 1) * bs + (long long)(gridDim.z - 1) * hs + (long long)(Nq - 1) * ld + Nk;
  const int D = Nq + Nk - 1;
  const int d0 = blockIdx.x * L * V;                             // diagonal index d: j = i + d - (Nq - 1)
  const int dl = d0 + lane * V - (Nq - 1);
  // rows that meet this strip: 0 <= i + d - (Nq - 1) < Nk for some d of it
  const int lo = max(max(ck * rows, Nq - 1 - (d0 + L * V - 1)), 0), hi = min(min((ck + 1) * rows, Nq), Nk + Nq - 1 - d0);
  float acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
  for (long long b = b0; b < b1; ++b) {
    const long long at = b * bs + (long long)h * hs;
    for (int i = lo + grp; i < hi; i += RG * U) {
      Raw8<T> v[U];
      const bool inside = i + d0 - (Nq - 1) >= 0 && i + RG * (U - 1) + d0 - (Nq - 1) + L * V <= Nk && i + RG * (U - 1) < hi;
      if (inside) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u].load_all(g + at + (i + RG * u) * ld + (i + RG * u + dl), true);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += v[u].at(e);
      } else {
        bool alone[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = i + RG * u, j = r + dl;
          const long long o = at + r * ld + j;
          const bool any = r < hi && j > -V && j < Nk;
          alone[u] = any && (o < 0 || o + V > span);
          v[u].load_all(g + o, any && !alone[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int j = i + RG * u + dl;
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += (unsigned)(j + e) < (unsigned)Nk ? v[u].at(e) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (alone[u]) {
            const int r = i + RG * u, j = r + dl;
            const T* p = g + at + r * ld + j;
#pragma unroll
            for (int e = 0; e < V; ++e)
              if ((unsigned)(j + e) < (unsigned)Nk) acc[e] += (float)p[e];
          }
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) buf[grp][lane * V + e] = acc[e];
  edge[threadIdx.x] = mine;
  __syncthreads();
  for (int k = threadIdx.x; k < L * V; k += 256) {
    float t = buf[0][k];
#pragma unroll
    for (int w = 1; w < RG; ++w) t += buf[w][k];
    buf[0][k] = t;
  }
  __syncthreads();
  const int buckets = (borders.n + 1) * (both ? 2 : 1), end = D - d0 < L * V ? D - d0 : L * V;
  float* line = part + ((long long)blockIdx.y * gridDim.x + blockIdx.x) * buckets * gridDim.z + h;
  for (int bk = threadIdx.x >> 4; bk < buckets; bk += 16) {
    long long r0, r1;
    bucket_run(bk, edge, borders.n, both, r0, r1);
    const long long shift = (long long)(Nq - 1) + off - d0;      // r = j - i - off lies on the strip's diagonal r + shift
    const int k0 = (int)min(max(r0 + shift, 0ll), (long long)end), k1 = (int)min(max(r1 + shift, 0ll), (long long)end);
    float t = 0.f;
    for (int k = k0 + (threadIdx.x & 15); k < k1; k += 16) t += buf[0][k];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) t += __shfl_xor(t, o, 16);
    if ((threadIdx.x & 15) == 0) line[(long long)bk * gridDim.z] = t;
  }
}

// Windows: sum over a run of the batch, element by element (grid: pieces of the [H, N, N] plane, batch chunks), then over the pairs of each
// bucket.  The four wavefronts of a workgroup take the same 64 vectors and a quarter of the run each, so that a line of sums is written and read
// again for four times as much of the batch.
template <typename T>
__global__ void __launch_bounds__(256)
window_bias_sum_kernel(const T* __restrict__ g, long long bs, long long hs, long long ld, float* __restrict__ part, int H, int N, int nvec,
                       long long B, long long chunk) {
  const long long span = (B - 1) * bs + (long long)(H - 1) * hs + (long long)(N - 1) * ld + N;
  __shared__ float buf[3][64][9];
  const int lane = threadIdx.x & 63, grp = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long all = (long long)H * N * nvec, at = (long long)blockIdx.x * 64 + lane, i = at < all ? at : all - 1;
  const int v = (int)(i % nvec);
  const long long hr = i / nvec;
  const int row = (int)(hr % N), h = (int)(hr / N), n = N - v * 8;
  const long long b0 = (long long)blockIdx.y * chunk, b1 = b0 + chunk < B ? b0 + chunk : B;
  const T* p = g + h * hs + row * ld + v * 8;
  float acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  // what a row's last lane reads beyond it lies in the tensor up to the last batch entries, and is not stored
  const long long here = (long long)h * hs + (long long)row * ld + v * 8;
  long long bv = b1;
  if (n < 8) {
    while (bv > b0 && here + (bv - 1) * bs + 8 > span) --bv;     // a step or two, or all where the batch is one entry broadcast
  }
  long long b = b0 + grp;
#pragma unroll 4
  for (; b < bv; b += 4) {
    Raw8<T> x;
    x.load_all(p + b * bs, true);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += x.at(e);
  }
  for (; b < b1; b += 4) {
    float x[8];
    load8(p + b * bs, n, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += x[e];
  }
  if (grp)
#pragma unroll
    for (int e = 0; e < 8; ++e) buf[grp - 1][lane][e] = acc[e];
  __syncthreads();
  if (grp || at >= all) return;
#pragma unroll
  for (int w = 0; w < 3; ++w)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += buf[w][lane][e];
  store8(part + (((long long)blockIdx.y * H + h) * N + row) * N + v * 8, n, acc);
}

// The sums come in `lines` parts (few: with more a launch adds them up first).  A workgroup takes the pairs of one vertical offset and head: a lane the pairs (xi, xj), whose rows of ws elements it adds over the token rows
// yj, then one of the 2 ws - 1 horizontal offsets each.
__global__ void __launch_bounds__(256)
window_bias_finish_kernel(const float* __restrict__ sum, int lines, float* __restrict__ dtable, int H, int ws) {
  extern __shared__ float pair[];                                // [xi][xj]
  const int h = blockIdx.y, N = ws * ws, w = 2 * ws - 1, dy = (int)blockIdx.x - (ws - 1);          // yi - yj
  const int y0 = max(0, -dy), y1 = min(ws, ws - dy);             // yj
  for (int t = threadIdx.x; t < N; t += 256) {
    const int xi = t / ws, xj = t - xi * ws;
    float s = 0.f;
    for (int l = 0; l < lines; ++l)
#pragma unroll 4
      for (int yj = y0; yj < y1; ++yj) s += sum[(((long long)l * H + h) * N + (yj + dy) * ws + xi) * N + yj * ws + xj];
    pair[t] = s;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < w; k += 256) {
    const int dx = k - (ws - 1), x0 = max(0, -dx), x1 = min(ws, ws - dx);
    float s = 0.f;
    for (int xj = x0; xj < x1; ++xj) s += pair[(xj + dx) * ws + xj];
    dtable[((long long)blockIdx.x * w + k) * H + h] = s;
  }
}

// Workgroups: about ten a CU (8 x 8 x 1023^2 bf16 34.5 us; six 41, sixteen 36.5; 16384^2 fp16 124, 154, 132); a long sequence's rows are split, a large batch's entries go several to one.
// Few rows and entries: one workgroup a head takes them all, and no second launch adds up lines (4 x 6 x 47 x 47: 10 us in two launches).
struct SeqShape { int lanes, strips, chunks, rows; long long bper, lines; };
inline SeqShape seq_shape(long long B, int H, int Nq, int Nk) {
  SeqShape s;
  for (int lanes = 8; lanes <= 64; lanes *= 2) {
    const int pass = rows_in_flight(lanes) * (256 / lanes);
    if ((long long)Nq + Nk - 1 <= 8 * lanes && B * ((Nq + pass - 1) / pass) <= 6) return {lanes, 1, 1, Nq, B, 1};
  }
  s.lanes = Nk >= 512 ? 64 : Nk >= 256 ? 32 : Nk >= 128 ? 16 : 8;
  s.strips = (int)(((long long)Nq + Nk - 1 + 8 * s.lanes - 1) / (8 * s.lanes));
  const long long per = B * H * s.strips;
  long long want = (2560 + per - 1) / per;
  const long long most = (Nq + 2048 / s.lanes - 1) / (2048 / s.lanes);              // eight passes of rows at least
  if (want > most) want = most;
  const int pass = rows_in_flight(s.lanes) * (256 / s.lanes);
  s.rows = ((int)((Nq + want - 1) / want) + pass - 1) / pass * pass;               // whole passes
  s.chunks = (Nq + s.rows - 1) / s.rows;
  s.bper = per > 2560 ? (per + 2559) / 2560 : 1;
  s.lines = (B + s.bper - 1) / s.bper * s.chunks;
  return s;
}
struct WinShape { long long chunk; int chunks; };
inline WinShape win_shape(long long B, int H, int N) {
  const long long blocks = ((long long)H * N * ((N + 7) / 8) + 63) / 64;
  long long want = (2048 + blocks - 1) / blocks;
  const long long most = (B + 31) / 32;                          // eight windows a wavefront (58 x 10 x 196^2 bf16: 17.6 us, with four 20.0 us)
  if (want > most) want = most;
  if (want > 65535) want = 65535;
  WinShape s;
  s.chunk = (B + want - 1) / want;
  s.chunks = (int)((B + s.chunk - 1) / s.chunk);
  return s;
}

inline int fill_borders(Borders& b, const int* borders_host, int n) {
  if (n < 0 || n > kMaxBuckets || (n && !borders_host)) return fail(OVIS_EINVAL, "relpos_bias: 0 to %d borders", kMaxBuckets);
  b.n = n;
  for (int i = 0; i < n; ++i) {
    b.at[i] = borders_host[i];
    if (b.at[i] < 1 || (i && b.at[i] < b.at[i - 1])) return fail(OVIS_EINVAL, "relpos_bias: borders must be positive and ascending");
  }
  return OVIS_OK;
}

}  // namespace

#define RP_TYPE(dtype, CALL)                         \
  if (dtype == OVIS_F32) { CALL(float) }             \
  else if (dtype == OVIS_F16) { CALL(_Float16) }     \
  else { CALL(__bf16) }

extern "C" int ovis_relpos_bias_1d(const float* table, void* out, const int* borders_host, int nborders, int bidirectional, int H, int Nq, int Nk,
                                   int ld, long long q_offset, int dtype, ovis_stream_t stream) {
  OVIS_REQUIRE(table && out && ovis::dtype_ok(dtype), "relpos_bias_1d: null pointer or type %d", dtype);
  OVIS_REQUIRE(H > 0 && H <= 65535 && Nq > 0 && Nk > 0 && Nq < (1 << 30) && Nk < (1 << 30) && q_offset < (1ll << 60) && q_offset > -(1ll << 60),
               "relpos_bias_1d: H %d, Nq %d, Nk %d", H, Nq, Nk);
  OVIS_REQUIRE(ld >= Nk && ld % (16 / ovis::dtype_size(dtype)) == 0 && ((uintptr_t)out & 15) == 0,
               "relpos_bias_1d: rows of 16-byte multiples at 16-byte addresses");
  Borders b;
  const int rc = fill_borders(b, borders_host, nborders);
  if (rc != OVIS_OK) return rc;
  const int cols = 256 * 16 / ovis::dtype_size(dtype);
  const unsigned strips = ovis::cdiv(ld, cols);
  int rows = 64;
  while ((long long)((Nq + rows - 1) / rows) > 65535) rows *= 2;
  OVIS_REQUIRE(rows <= 8192, "relpos_bias_1d: too many rows");
#define RP_GO(T)                                                                                                                            \
  hipLaunchKernelGGL((relpos_fwd_kernel<T>), dim3(strips, (Nq + rows - 1) / rows, H), dim3(256), (cols + rows) * sizeof(T),                 \
                     (hipStream_t)stream, table, (T*)out, b, bidirectional, H, Nq, Nk, ld, q_offset, rows);
  RP_TYPE(dtype, RP_GO)
#undef RP_GO
  return ovis::check_launch("relpos_bias_1d");
}

extern "C" long long ovis_relpos_bias_1d_backward_workspace_bytes(long long B, int H, int Nq, int Nk, int buckets) {
  if (B <= 0 || H <= 0 || Nq <= 0 || Nk <= 0 || buckets <= 0) return 0;
  const SeqShape s = seq_shape(B, H, Nq, Nk);
  return s.lines * s.strips * H * buckets * 4;
}

extern "C" int ovis_relpos_bias_1d_backward(const void* dbias, long long bs, long long hs, long long ld, float* dtable, float* workspace,
                                            const int* borders_host, int nborders, int bidirectional, long long B, int H, int Nq, int Nk,
                                            long long q_offset, int dtype, ovis_stream_t stream) {
  OVIS_REQUIRE(dbias && dtable && workspace && ovis::dtype_ok(dtype), "relpos_bias_1d_backward: null pointer or type %d", dtype);
  OVIS_REQUIRE(B > 0 && H > 0 && H <= 65535 && Nq > 0 && Nk > 0 && Nq < (1 << 30) && Nk < (1 << 30) && q_offset < (1ll << 60) &&
               q_offset > -(1ll << 60), "relpos_bias_1d_backward: B %lld, H %d, Nq %d, Nk %d", B, H, Nq, Nk);
  OVIS_REQUIRE(ld >= 0 && bs >= 0 && hs >= 0, "relpos_bias_1d_backward: negative stride");
  Borders b;
  const int rc = fill_borders(b, borders_host, nborders);
  if (rc != OVIS_OK) return rc;
  const SeqShape s = seq_shape(B, H, Nq, Nk);
  const int buckets = (b.n + 1) * (bidirectional ? 2 : 1), W = buckets * H;                               // at most 514 x 65535
  const long long parts = s.lines * s.strips;
  OVIS_REQUIRE(s.lines <= 65535 && s.strips <= ovis::kMostBlocks && parts < (1ll << 31) && (long long)H * (Nq + Nk - 1) < (1ll << 31),
               "relpos_bias_1d_backward: B %lld, H %d, Nq %d, Nk %d are too large for one call", B, H, Nq, Nk);
  float* to = parts > 1 ? workspace : dtable;
#define RP_LANES(T)                                                                                                                         \
  if (s.lanes == 64) { RP_GO(T, 64) } else if (s.lanes == 32) { RP_GO(T, 32) } else if (s.lanes == 16) { RP_GO(T, 16) } else { RP_GO(T, 8) }
#define RP_GO(T, L)                                                                                                                         \
  hipLaunchKernelGGL((relpos_bwd_kernel<T, L>), dim3(s.strips, (unsigned)s.lines, H), dim3(256), 0, (hipStream_t)stream, (const T*)dbias, bs,  \
                     hs, ld, to, b, bidirectional, q_offset, B, s.bper, Nq, Nk, s.rows, s.chunks);
  RP_TYPE(dtype, RP_LANES)
#undef RP_LANES
#undef RP_GO
  const int launched = ovis::check_launch("relpos_bias_1d_backward");
  if (launched != OVIS_OK || parts == 1) return launched;
  return ovis::column_sum_finish(workspace, (int)parts, W, dtable, W, dtable, (hipStream_t)stream);
}

extern "C" long long ovis_swin_relpos_bias_backward_workspace_bytes(long long B, int H, int ws) {
  if (B <= 0 || H <= 0 || ws <= 0 || ws > 64) return 0;
  return ((long long)win_shape(B, H, ws * ws).chunks + 1) * H * ws * ws * ws * ws * 4;
}

extern "C" int ovis_swin_relpos_bias_backward(const void* dbias, long long bs, long long hs, long long ld, float* dtable, float* workspace,
                                              long long B, int H, int ws, int dtype, ovis_stream_t stream) {
  OVIS_REQUIRE(dbias && dtable && workspace && ovis::dtype_ok(dtype), "swin_relpos_bias_backward: null pointer or type %d", dtype);
  OVIS_REQUIRE(B > 0 && H > 0 && H <= 65535 && ws > 0 && ws <= 64 && ld >= 0 && bs >= 0 && hs >= 0,
               "swin_relpos_bias_backward: B %lld, heads %d, window %d (1 to 64)", B, H, ws);
  const int N = ws * ws, nvec = (N + 7) / 8;
  const WinShape s = win_shape(B, H, N);
  const long long W = (long long)H * N * N;
  OVIS_REQUIRE(W < (1ll << 31), "swin_relpos_bias_backward: %d heads of windows of %d are too large for one call", H, ws);
#define RP_GO(T)                                                                                                                            \
  hipLaunchKernelGGL((window_bias_sum_kernel<T>), dim3(ovis::cdiv((long long)H * N * nvec, 64), s.chunks), dim3(256), 0,                   \
                     (hipStream_t)stream, (const T*)dbias, bs, hs, ld, workspace + W, H, N, nvec, B, s.chunk);
  RP_TYPE(dtype, RP_GO)
#undef RP_GO
  int rc = ovis::check_launch("swin_relpos_bias_backward");
  const bool few = s.chunks <= 4;
  if (rc == OVIS_OK && !few)
    rc = ovis::column_sum_finish(workspace + W, s.chunks, (int)W, workspace, (int)W, workspace, (hipStream_t)stream);
  if (rc != OVIS_OK) return rc;
  hipLaunchKernelGGL(window_bias_finish_kernel, dim3(2 * ws - 1, H), dim3(256), N * 4, (hipStream_t)stream,
                     few ? workspace + W : workspace, few ? s.chunks : 1, dtable, H, ws);
  return ovis::check_launch("swin_relpos_bias_backward");
}
