// What follows the products of the forward pass, for eight neighbouring
// columns of one row: bias, what training keeps, activation, gate, residual
// and the one rounding to the type.
#pragma once

#include "feed_forward.h"
#include "linear.h"

namespace ff {

enum Keep { kNothing = 0, kPre = 1, k8 = 2 };

// columns n.. of the bias, zeros behind the last one
template <typename T>
__device__ __forceinline__ Vec8<T> bias8(const Forward& f, long n, long half) {
  if (f.bias == nullptr) return Vec8<T>{};
  return some8((const T*)f.bias + half + n, f.n - n);
}

// Codes and exponent of eight pre-activations, columns n..; the lanes X, Y and
// X + Y away hold the rest of a group of 32 columns.
template <int X, int Y>
__device__ __forceinline__ uint2 codes8(const Forward& f, long n,
                                        const float* v, int& e) {
  float w[8];
  const bool whole = n + 8 <= f.n;
#pragma unroll
  for (int k = 0; k < 8; k++) w[k] = whole || n + k < f.n ? v[k] : 0.f;
  return encode8<X, Y>(w, e);
}

// Keeps eight pre-activations of row m, columns n.. of the gated layer's up
// half or the other.
template <typename T, int KEEP, bool GATED, int X, int Y>
__device__ __forceinline__ void keep_pre(const Forward& f, long m, long n,
                                         bool up, bool live, const float* v) {
  const long at = m * f.ldp + (up ? f.ldp / 2 : 0) + n;
  if constexpr (KEEP == kPre) {
    if (live && n < f.n) {
      if constexpr (GATED) {
        u16x8 hi;
        *(uint2*)(f.low + at) = split24(v, hi);
        *(u16x8*)((unsigned short*)f.pre + at) = hi;
      } else {
        *(Vec8<T>*)((T*)f.pre + at) = to8<T>(v);
      }
    }
  } else if constexpr (KEEP == k8) {
    int e;
    const uint2 codes = codes8<X, Y>(f, n, v, e);
    if (live && (n & ~31L) < f.n) {
      *(uint2*)(f.codes + at) = codes;
      if ((n & 31) == 0) f.scales[at >> 5] = (unsigned char)(e + 127);
    }
  }
}

template <int ACT>
__device__ __forceinline__ void act8(float* v, int) {
#pragma unroll
  for (int k = 0; k < 8; k++) v[k] = act<ACT>(v[k]);
}
// ACT < 0: `a` says which
template <>
__device__ __forceinline__ void act8<-1>(float* v, int a) {
  if (a == kGelu) act8<kGelu>(v, a);
  else if (a == kSilu) act8<kSilu>(v, a);
  else if (a == kRelu) act8<kRelu>(v, a);
}

// Eight columns of the residual, zeros where there is none.
template <typename T>
__device__ __forceinline__ Vec8<T> residual8(const Forward& f, long m, long n) {
  if (f.res == nullptr || m >= f.m) return Vec8<T>{};
  return some8((const T*)f.res + m * f.ldr + n, f.n - n);
}

// v (and the gated layer's u): the products, with the bias; r: the residual.
// All lanes of a group come here, `live` or not.
template <typename T, int KEEP, int ACT, bool GATED, int X, int Y>
__device__ __forceinline__ void finish8(const Forward& f, long m, long n,
                                        bool live, float* v, float* u,
                                        Vec8<T> r) {
  keep_pre<T, KEEP, GATED, X, Y>(f, m, n, false, live, v);
  if constexpr (GATED) keep_pre<T, KEEP, GATED, X, Y>(f, m, n, true, live, u);
  act8<ACT>(v, f.act);
#pragma unroll
  for (int k = 0; k < 8; k++) {
    if constexpr (GATED) v[k] *= u[k];
    else v[k] += (float)r[k];
  }
  if (!live || n >= f.n) return;
  store_some((T*)f.y + m * f.n + n, f.n - n, v);
}

}  // namespace ff
