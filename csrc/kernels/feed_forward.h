// What the feed-forward kernels share: activations with their slopes, the
// forms that pre-activations are kept in, and vectors of 16-bit values.
#pragma once

#include "common.h"

namespace ff {

enum Act { kNone = 0, kRelu = 1, kGelu = 2, kSilu = 3 };

using f32x8 = __attribute__((ext_vector_type(8))) float;

// 1 / (1 + exp(-v)); exact limits at both ends
__device__ __forceinline__ float sigmoid(float v) {
  return __builtin_amdgcn_rcpf(
      1.f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f));
}

// tanh form: 0.5 v (1 + tanh u) = v sigmoid(2u), u = c (v + a v^3)
constexpr float kGelu2C = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

template <int a>
__device__ __forceinline__ float act(float v) {
  if (a == kGelu) return v * sigmoid(kGelu2C * (v + kGeluA * v * v * v));
  if (a == kSilu) return v * sigmoid(v);
  if (a == kRelu) return v < 0.f ? 0.f : v;  // NaN stays
  return v;
}

// d act / dv.  Past |v| = 12 the tanh form's slope is 0 or 1 to fp32; the
// comparisons hold v there, so that v^3 stays finite, and pass NaN on.
template <int a>
__device__ __forceinline__ float slope(float v) {
  if (a == kGelu) {
    v = v > 12.f ? 12.f : v;
    v = v < -12.f ? -12.f : v;
    const float z = sigmoid(kGelu2C * (v + kGeluA * v * v * v));
    return z + v * z * (1.f - z) * kGelu2C * (1.f + 3.f * kGeluA * v * v);
  }
  if (a == kSilu) {
    const float z = sigmoid(v);
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

__device__ __forceinline__ bool is_finite(float v) {
  return __builtin_fabsf(v) <= 3.402823466e38f;
}

__device__ __forceinline__ int scale_exp(float amax) {
  const unsigned b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 135 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < -118 ? -118 : (e > 120 ? 120 : e);
}

__device__ __forceinline__ float two_to(int e) {
  return __uint_as_float((unsigned)(e + 127) << 23);
}

__device__ __forceinline__ uint2 encode8(const float* v, int e) {
  const float s = two_to(-e);
  float u[8];
#pragma unroll
  for (int k = 0; k < 8; k++)
    u[k] = is_finite(v[k]) ? v[k] * s : __uint_as_float(0x7fc00000u);
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(u[0], u[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(u[2], u[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(u[4], u[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(u[6], u[7], hi, true);
  return make_uint2((unsigned)lo, (unsigned)hi);
}

__device__ __forceinline__ void decode8(uint2 c, unsigned char scale,
                                        float* v) {
  const float s = two_to((int)scale - 127);
  using f32x2 = __attribute__((ext_vector_type(2))) float;
  f32x2 p;
  p = __builtin_amdgcn_cvt_pk_f32_fp8(c.x, false);
  v[0] = p[0] * s, v[1] = p[1] * s;
  p = __builtin_amdgcn_cvt_pk_f32_fp8(c.x, true);
  v[2] = p[0] * s, v[3] = p[1] * s;
  p = __builtin_amdgcn_cvt_pk_f32_fp8(c.y, false);
  v[4] = p[0] * s, v[5] = p[1] * s;
  p = __builtin_amdgcn_cvt_pk_f32_fp8(c.y, true);
  v[6] = p[0] * s, v[7] = p[1] * s;
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

// ---- 16-bit vectors --------------------------------------------------------

template <typename T> using Vec8 = __attribute__((ext_vector_type(8))) T;

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* v) {
  const Vec8<T> u = *(const Vec8<T>*)p;
#pragma unroll
  for (int k = 0; k < 8; k++) v[k] = (float)u[k];
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* v) {
  Vec8<T> u;
#pragma unroll
  for (int k = 0; k < 8; k++) u[k] = (T)v[k];
  *(Vec8<T>*)p = u;
}

// n valid values from an address of any alignment, zeros behind them
template <typename T>
__device__ __forceinline__ void load_some(const T* p, long n, float* v) {
#pragma unroll
  for (int k = 0; k < 8; k++) v[k] = k < n ? (float)p[k] : 0.f;
}

template <typename T>
__device__ __forceinline__ void store_some(T* p, long n, const float* v) {
#pragma unroll
  for (int k = 0; k < 8; k++)
    if (k < n) p[k] = (T)v[k];
}

__device__ __forceinline__ void store24(unsigned short* hi, unsigned char* lo,
                                        const float* v) {
  u16x8 h;
  unsigned l[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const unsigned b = to_24(v[k]);
    h[k] = (unsigned short)(b >> 8);
    l[k >> 2] |= (b & 255u) << (k & 3) * 8;
  }
  *(u16x8*)hi = h;
  *(uint2*)lo = make_uint2(l[0], l[1]);
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
