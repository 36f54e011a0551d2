// Element types, unaligned 8-element vectors and the 8-bit block format of the training-side operators (gfx950 only).
//
// Types: OVIS_F32 / OVIS_F16 / OVIS_BF16 tensors; all arithmetic is f32 and each output is rounded once (to nearest even).
// A lane moves 8 consecutive elements; rows need no alignment beyond the element's own (the hardware takes 16-byte global accesses at any
// address), so odd row lengths and strided views use the same vector accesses as aligned ones and only a row's last lane goes by elements.
//
// 8-bit block format: e4m3 codes and one power-of-two scale (e8m0: 2^(byte - 127)) per 32 columns of a row.  Four neighbouring lanes hold a
// block.  The scale is the smallest power of two in [2^-100, 2^120] under which the block's largest finite magnitude is at most 448, so no
// value saturates and every value above 2^-6 of its scale is off by at most 2^-4 of itself.  The limits keep scale, value and their product
// inside f32's normal range.  e4m3 has no infinity: infinities and NaN become the NaN code (-infinity in front of a ReLU: -0) and do not take part
// in the block's maximum.
// (Values from 2^128 (1 - 2^-5) on round to a code that stands for 2^128, an infinity in f32.)
#pragma once
#include "common.h"

namespace ovis {

template <typename T> struct Vec8Of;                     // 8 elements, aligned as one element
typedef _Float16 f16x8_u __attribute__((ext_vector_type(8), aligned(2)));
typedef __bf16 bf16x8_u __attribute__((ext_vector_type(8), aligned(2)));
typedef float f32x8_u __attribute__((ext_vector_type(8), aligned(4)));
template <> struct Vec8Of<_Float16> { using type = f16x8_u; };
template <> struct Vec8Of<__bf16> { using type = bf16x8_u; };
template <> struct Vec8Of<float> { using type = f32x8_u; };
typedef unsigned u32x2_u __attribute__((ext_vector_type(2), aligned(1)));

// n (1..8) elements of p into v, the others 0.  Here and below a row's last elements are read at indexes held at n - 1, without conditions, so that
// the reads are in flight together: one condition each makes the compiler wait for each.
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, int n, float (&v)[8]) {
  if (n >= 8) {
    const typename Vec8Of<T>::type t = *reinterpret_cast<const typename Vec8Of<T>::type*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)t[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)p[e < n ? e : n - 1];
#pragma unroll
    for (int e = 1; e < 8; ++e) v[e] = e < n ? v[e] : 0.f;
  }
}

// the same where `on` says that eight elements can be read: what follows a row's end is the next rows', and becomes 0
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, int n, bool on, float (&v)[8]) {
  load8(p, on ? 8 : n, v);
#pragma unroll
  for (int e = 1; e < 8; ++e) v[e] = e < n ? v[e] : 0.f;
}

// the same, kept in the stored type
template <typename T>
struct Raw8 {
  typename Vec8Of<T>::type v;
  // n elements of a row at p, the others anything (n <= 0: 0).  on: the eight lie in the tensor even where the row ends earlier (the next rows
  // follow): they are read as one vector, which nothing waits for
  __device__ __forceinline__ void load(const T* __restrict__ p, int n, bool on) {
    v = (typename Vec8Of<T>::type)0;
    if (n > 0) {
      if (n >= 8 || on) {
        v = *reinterpret_cast<const typename Vec8Of<T>::type*>(p);
      } else {
        T t[7];
#pragma unroll
        for (int e = 0; e < 7; ++e) t[e] = p[e < n ? e : n - 1];
#pragma unroll
        for (int e = 0; e < 7; ++e) v[e] = t[e];
      }
    }
  }
  __device__ __forceinline__ void load_all(const T* __restrict__ p, bool any) {       // all eight, or none
    v = (typename Vec8Of<T>::type)0;
    if (any) v = *reinterpret_cast<const typename Vec8Of<T>::type*>(p);
  }
  __device__ __forceinline__ float at(int e) const { return (float)v[e]; }
  // the compiler takes the registers as new from here on, so that it widens them again where they are used instead of keeping both forms
  __device__ __forceinline__ void hide() {
    typedef unsigned words __attribute__((ext_vector_type(sizeof(v) / 4)));
    words w = __builtin_bit_cast(words, v);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(v) / 4); ++i) asm volatile("" : "+v"(w[i]));
    v = __builtin_bit_cast(typename Vec8Of<T>::type, w);
  }
};

template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, int n, const float (&v)[8]) {
  if (n >= 8) {
    typename Vec8Of<T>::type t;
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = (T)v[e];
    *reinterpret_cast<typename Vec8Of<T>::type*>(p) = t;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = (T)v[e];
  }
}

__device__ __forceinline__ float pow2f(int e) { return __builtin_bit_cast(float, (unsigned)(e + 127) << 23); }   // -126 <= e <= 127

// maximum over the four lanes of a block (quad_perm moves inside groups of four lanes: no LDS)
__device__ __forceinline__ unsigned quad_max(unsigned a) {
  a = max(a, (unsigned)__builtin_amdgcn_mov_dpp((int)a, 0xB1, 0xf, 0xf, true));            // lanes 1 0 3 2
  return max(a, (unsigned)__builtin_amdgcn_mov_dpp((int)a, 0x4E, 0xf, 0xf, true));         // lanes 2 3 0 1
}

__device__ __forceinline__ unsigned magnitude(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

// 8 values of one lane (the block's other 24 in its three neighbours; all four lanes active) -> 8 codes, and the scale's byte.
// signed_zero: a value of 0 gets the code -0, so that a code's sign bit says "not positive" (ReLU's derivative).  So does -infinity, whose ReLU
// and whose derivative are 0 like those of any value below 0: as a NaN it would come back where the forward pass gave 0.
// The maximum is taken over the magnitudes' bits: they order as the values do, with infinity and then every NaN (signalling ones too, which
// a floating-point maximum would pass on) at the top.
__device__ __forceinline__ u32x2_u encode8(const float (&v)[8], bool signed_zero, unsigned& scale_byte) {
  constexpr unsigned kInf = 0x7f800000u;
  unsigned a = 0u;
#pragma unroll
  for (int e = 0; e < 8; ++e) a = max(a, magnitude(v[e]));
  a = quad_max(a);
  float w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = v[e];
  u32x2_u keep = {~0u, ~0u};
  if (a >= kInf) {                                                 // rare: the maximum of the finite ones, the others to NaN
    a = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool fine = magnitude(w[e]) < kInf;
      a = max(a, fine ? magnitude(w[e]) : 0u);
      w[e] = fine ? w[e] : signed_zero && v[e] < 0.f ? -0.f : NAN;
      if (w[e] != w[e]) keep[e >> 2] &= ~(0x80u << (8 * (e & 3)));  // the conversion sets a NaN's sign, which is for "not positive" alone
    }
    a = quad_max(a);
  }
  int s = (int)(a >> 23) - 135 + ((a & 0x7fffffu) > 0x600000u ? 1 : 0);             // 1.75 * 2^8 = 448
  s = min(max(s, -100), 120);
  scale_byte = (unsigned)(s + 127);
  const float f = pow2f(-s);
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = signed_zero && w[e] == 0.f ? -0.f : w[e] * f;
  u32x2_u r;
  int t = __builtin_amdgcn_cvt_pk_fp8_f32(w[0], w[1], 0, false);
  t = __builtin_amdgcn_cvt_pk_fp8_f32(w[2], w[3], t, true);
  r[0] = (unsigned)t;
  t = __builtin_amdgcn_cvt_pk_fp8_f32(w[4], w[5], 0, false);
  t = __builtin_amdgcn_cvt_pk_fp8_f32(w[6], w[7], t, true);
  r[1] = (unsigned)t;
  r[0] &= keep[0], r[1] &= keep[1];
  return r;
}

// 8 codes -> the values they stand for (exact: 4 significant bits times a power of two)
__device__ __forceinline__ void decode8(u32x2_u c, unsigned scale_byte, float (&v)[8]) {
  const float f = pow2f((int)scale_byte - 127);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    v[4 * h] = __builtin_amdgcn_cvt_f32_fp8((int)c[h], 0) * f;
    v[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8((int)c[h], 1) * f;
    v[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8((int)c[h], 2) * f;
    v[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8((int)c[h], 3) * f;
  }
}

__device__ __forceinline__ void hide(u32x2_u& c) {
  unsigned a = c[0], b = c[1];
  asm volatile("" : "+v"(a), "+v"(b));
  c[0] = a, c[1] = b;
}

__device__ __forceinline__ u32x2_u load_codes(const uint8_t* __restrict__ p, int n) {
  u32x2_u c;
  if (n >= 8) {
    c = *reinterpret_cast<const u32x2_u*>(p);
  } else {
    c[0] = c[1] = 0u;
    if (n > 0) {
      unsigned t[7];
#pragma unroll
      for (int e = 0; e < 7; ++e) t[e] = p[e < n ? e : n - 1];
#pragma unroll
      for (int e = 0; e < 7; ++e) c[e >> 2] |= e < n ? t[e] << (8 * (e & 3)) : 0u;
    }
  }
  return c;
}

// the same, with the codes behind the row's end where `on` says that they can be read
__device__ __forceinline__ u32x2_u load_codes(const uint8_t* __restrict__ p, int n, bool on) { return load_codes(p, n > 0 && on ? 8 : n); }

__device__ __forceinline__ void store_codes(uint8_t* __restrict__ p, int n, u32x2_u c) {
  if (n >= 8) {
    *reinterpret_cast<u32x2_u*>(p) = c;
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) p[e] = (uint8_t)(c[e >> 2] >> (8 * (e & 3)));
  }
}

// sums the P lines of part [P][W] in a fixed order: columns below `split` to out0, the others to out1 (layernorm_train.hip)
struct ColumnSum { const float* part; int P, W; float* out0; int split; float* out1; };
int column_sum_two(const ColumnSum& a, const ColumnSum& b, hipStream_t stream);         // two of them in one launch
int column_sum_finish(const float* part, int P, int W, float* out0, int split, float* out1, hipStream_t stream);

// a launch's lanes along a dimension are counted in 32 bits: so many workgroups of 256 lanes at most
constexpr long long kMostBlocks = (1ll << 24) - 1;

inline bool dtype_ok(int t) { return t == OVIS_F32 || t == OVIS_F16 || t == OVIS_BF16; }
inline int dtype_size(int t) { return t == OVIS_F32 ? 4 : 2; }

}  // namespace ovis
