// Activations in 8 bits back to values, for act8.hip and for the backward
// pass, which does it in its first launch.
#pragma once

#include "feed_forward.h"
#include "linear.h"

namespace ff {

template <typename T> struct Most;
template <> struct Most<__bf16> { static constexpr float v = 3.38953139e38f; };
template <> struct Most<_Float16> { static constexpr float v = 65504.f; };
template <> struct Most<float> { static constexpr float v = 3.402823466e38f; };

// Eights of values `first`, `first` + `step`, ...
template <typename T>
__device__ __forceinline__ void unpack_values(const Pack& p, long first,
                                              long step) {
  const long per = (p.ldx + 7) / 8, total = p.m * per;
  for (long i = first; i < total; i += step) {
    const long r = i / per, c = (i - r * per) * 8;
    float v[8] = {};
    if (c < p.n) {  // codes behind n, up to the multiple of 32, are zeros
      const long at = r * p.ldc + c;
      decode8(*(const uint2*)(p.codes + at), p.scales[at >> 5], v);
    }
    // The largest magnitudes may round up past the type's range: they are
    // held at its largest value.  NaN fails both comparisons and stays.
#pragma unroll
    for (int k = 0; k < 8; k++) {
      v[k] = v[k] > Most<T>::v ? Most<T>::v : v[k];
      v[k] = v[k] < -Most<T>::v ? -Most<T>::v : v[k];
    }
    T* x = (T*)p.x + r * p.ldx + c;
    if (p.vec)
      store8(x, v);
    else
      store_some(x, p.ldx - c, v);
  }
}

}  // namespace ff
