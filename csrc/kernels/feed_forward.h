// What the feed-forward kernels share: activations with their slopes, the
// forms that pre-activations are kept in, and vectors of 16-bit values.
#pragma once

#include "common.h"

namespace ff {

enum Act { kNone = 0, kRelu = 1, kGelu = 2, kSilu = 3 };

using f32x8 = __attribute__((ext_vector_type(8))) float;

// 1 / (1 + 2^-v); exact limits at both ends
__device__ __forceinline__ float sigmoid2(float v) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-v));
}

// tanh form: 0.5 v (1 + tanh u) = v sigmoid(2u), u = c (v + a v^3); here with
// the exponential's base 2: 2u log2(e) = v (kC + kA v^2).  It takes a fifth of
// the instructions of the tanh, which counts where a tile's 256 x 256 sums
// pass through one wave a SIMD.
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kC = 2.302208198144325f;    // 2 sqrt(2 / pi) log2(e)
constexpr float kA = 0.10294324142182365f;  // 0.044715 kC
constexpr float kGelu2C = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGelu6A = 0.21406445567880206f;  // 3 * 0.044715 * that

template <int a>
__device__ __forceinline__ float act(float v) {
  if (a == kGelu) return v * sigmoid2(v * __builtin_fmaf(v * v, kA, kC));
  if (a == kSilu) return v * sigmoid2(v * kLog2E);
  if (a == kRelu) return v < 0.f ? 0.f : v;  // NaN stays
  return v;
}

// d act / dv.  Past |v| = 12 the tanh form's slope is 0 or 1 to fp32, and past
// 100 silu's; the comparisons hold v there, so that v^3 and, where v was kept
// in fp16 and is infinite there, v itself stay finite, and pass NaN on.
template <int a>
__device__ __forceinline__ float slope(float v) {
  if (a == kGelu) {
    v = v > 12.f ? 12.f : v;
    v = v < -12.f ? -12.f : v;
    const float w = v * v;
    const float z = sigmoid2(v * __builtin_fmaf(w, kA, kC));
    return z + (1.f - z) * z * v * __builtin_fmaf(w, kGelu6A, kGelu2C);
  }
  if (a == kSilu) {
    v = v > 100.f ? 100.f : v;
    v = v < -100.f ? -100.f : v;
    const float z = sigmoid2(v * kLog2E);
    return z * (1.f + v * (1.f - z));
  }
  if (a == kRelu) return v > 0.f ? 1.f : 0.f;
  return 1.f;
}

// ---- activations in 8 bits -------------------------------------------------
//
// 32 neighbouring values share a power of two 2^e, the smallest with
// max |v| / 2^e <= 448 (e4m3's largest), and each is held as e4m3 of v / 2^e,
// rounded to nearest even.  e is kept as the byte e + 127, -118 <= e <= 120.
// A power of two makes both scalings exact: the one rounding is e4m3's own,
// at most 2^-4 of a value not below 2^-6 of the group's scale.  The largest
// is taken over the finite values; infinities and NaN are held as NaN.

// of the largest value's bits
__device__ __forceinline__ int scale_exp(unsigned b) {
  const int e = (int)(b >> 23) - 135 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < -118 ? -118 : (e > 120 ? 120 : e);
}

__device__ __forceinline__ float two_to(int e) {
  return __uint_as_float((unsigned)(e + 127) << 23);
}

// The larger of this lane's value and of that X lanes away (1, 2, 16 or 32).
template <int X>
__device__ __forceinline__ unsigned max_with(unsigned v) {
  unsigned a = v, b;
  if constexpr (X == 32) {
    const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    a = s[0], b = s[1];
  } else if constexpr (X == 16) {
    const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    a = s[0], b = s[1];
  } else {
    static_assert(X == 1 || X == 2, "lanes");
    constexpr int perm = X == 1 ? 0xb1 : 0x4e;  // of each four lanes
    b = __builtin_amdgcn_mov_dpp(v, perm, 0xf, 0xf, true);
  }
  return a > b ? a : b;
}

// Eight of a group's values, whose other 24 are in the lanes X, Y and X + Y
// away: their codes and the group's e.  Magnitudes are compared as whole
// numbers, in which infinities and NaN of either kind are the largest; where
// there is one, the finite values are looked for and the others made NaN.
template <int X, int Y>
__device__ __forceinline__ uint2 encode8(const float* v, int& e) {
  constexpr unsigned kInf = 0x7f800000u;
  float u[8];
  unsigned top = 0;
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const unsigned b = __float_as_uint(v[k]) & 0x7fffffffu;
    top = b > top ? b : top;
    u[k] = v[k];
  }
  top = max_with<Y>(max_with<X>(top));
  if (top >= kInf) {  // all four lanes or none
    top = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const unsigned b = __float_as_uint(v[k]) & 0x7fffffffu;
      if (b >= kInf) u[k] = __uint_as_float(0x7fc00000u);
      else top = b > top ? b : top;
    }
    top = max_with<Y>(max_with<X>(top));
  }
  e = scale_exp(top);
  const float s = two_to(-e);
#pragma unroll
  for (int k = 0; k < 8; k++) u[k] *= s;
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(u[0], u[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(u[2], u[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(u[4], u[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(u[6], u[7], hi, true);
  return make_uint2((unsigned)lo, (unsigned)hi);
}

__device__ __forceinline__ void decode4(unsigned c, unsigned char scale,
                                        float* v) {
  const float s = two_to((int)scale - 127);
  using f32x2 = __attribute__((ext_vector_type(2))) float;
  f32x2 p;
  p = __builtin_amdgcn_cvt_pk_f32_fp8(c, false);
  v[0] = p[0] * s, v[1] = p[1] * s;
  p = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
  v[2] = p[0] * s, v[3] = p[1] * s;
}

__device__ __forceinline__ void decode8(uint2 c, unsigned char scale,
                                        float* v) {
  decode4(c.x, scale, v);
  decode4(c.y, scale, v + 4);
}

// ---- pre-activations in 24 bits ---------------------------------------------
//
// The gated layer's gradient is a product of both its projections, and each
// rounded to 16 bits would add as much error to the gradients as their own
// rounding does.  They are kept as the upper 24 bits of float32 instead: the
// upper 16 in one plane, the next 8 in another.

__device__ __forceinline__ unsigned to_24(float v) {
  const unsigned b = __float_as_uint(v);
  return v != v ? 0x7fc000u : (b + 0x80u) >> 8;
}

__device__ __forceinline__ float from_24(unsigned hi, unsigned lo) {
  return __uint_as_float(hi << 16 | lo << 8);
}

using u16x8 = __attribute__((ext_vector_type(8))) unsigned short;
using u32x2 = __attribute__((ext_vector_type(2))) unsigned;

// ---- 16-bit vectors --------------------------------------------------------

template <typename T> using Vec8 = __attribute__((ext_vector_type(8))) T;

template <typename V>
__device__ __forceinline__ void widen(V u, float* v) {
#pragma unroll
  for (int k = 0; k < 8; k++) v[k] = (float)u[k];
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* v) {
  widen(*(const Vec8<T>*)p, v);
}

template <typename T>
__device__ __forceinline__ Vec8<T> to8(const float* v) {
  Vec8<T> u;
#pragma unroll
  for (int k = 0; k < 8; k++) u[k] = (T)v[k];
  return u;
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* v) {
  *(Vec8<T>*)p = to8<T>(v);
}

// n valid values from an address of any alignment, zeros behind them.  Eight
// are one access all the same, which the memory's units split where they have
// to: rows of odd lengths cost little more than others.
template <typename T>
using Any8 __attribute__((aligned(sizeof(T)))) = Vec8<T>;

template <typename T>
__device__ __forceinline__ Vec8<T> some8(const T* p, long n) {
  if (n >= 8) return *(const Any8<T>*)p;
  Vec8<T> u = {};
#pragma unroll
  for (int k = 0; k < 8; k++)
    if (k < n) u[k] = p[k];
  return u;
}

template <typename T>
__device__ __forceinline__ void load_some(const T* p, long n, float* v) {
  widen(some8(p, n), v);
}

template <typename T>
__device__ __forceinline__ void put_some(T* p, long n, Vec8<T> u) {
  if (n >= 8) {
    *(Any8<T>*)p = u;
  } else {
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (k < n) p[k] = u[k];
  }
}

template <typename T>
__device__ __forceinline__ void store_some(T* p, long n, const float* v) {
  put_some(p, n, to8<T>(v));
}

// the 16 upper bits of each, and the next 8 of all
__device__ __forceinline__ uint2 split24(const float* v, u16x8& hi) {
  unsigned l[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const unsigned b = to_24(v[k]);
    hi[k] = (unsigned short)(b >> 8);
    l[k >> 2] |= (b & 255u) << (k & 3) * 8;
  }
  return make_uint2(l[0], l[1]);
}

__device__ __forceinline__ void load24(const unsigned short* hi,
                                       const unsigned char* lo, float* v) {
  const u16x8 h = *(const u16x8*)hi;
  const uint2 l = *(const uint2*)lo;
#pragma unroll
  for (int k = 0; k < 8; k++)
    v[k] = from_24(h[k], ((k < 4 ? l.x : l.y) >> (k & 3) * 8) & 255u);
}

}  // namespace ff
