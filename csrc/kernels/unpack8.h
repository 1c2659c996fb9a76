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

// Runs of values `first`, `first` + `step`, ..., of 16 bytes each: eight
// values, four in fp32, whose eight would leave a lane in two stores that miss
// every other 16 bytes (8192 x 8192 takes 68 us so, and 92).
template <typename T>
__device__ __forceinline__ void unpack_values(const Pack& p, long first,
                                              long step) {
  constexpr int EACH = 16 / sizeof(T);
  const long per = (p.ldx + EACH - 1) / EACH, total = p.m * per;
  for (long i = first; i < total; i += step) {
    const long r = i / per, c = (i - r * per) * EACH;
    float v[EACH] = {};
    if (c < p.n) {  // codes behind n, up to the multiple of 32, are zeros
      const long at = r * p.ldc + c;
      if constexpr (EACH == 8)
        decode8(*(const uint2*)(p.codes + at), p.scales[at >> 5], v);
      else
        decode4(*(const unsigned*)(p.codes + at), p.scales[at >> 5], v);
    }
    // The largest magnitudes may round up past the type's range: they are
    // held at its largest value.  NaN fails both comparisons and stays.
#pragma unroll
    for (int k = 0; k < EACH; k++) {
      v[k] = v[k] > Most<T>::v ? Most<T>::v : v[k];
      v[k] = v[k] < -Most<T>::v ? -Most<T>::v : v[k];
    }
    T* x = (T*)p.x + r * p.ldx + c;
    if constexpr (EACH == 8) {
      if (p.vec)
        store8(x, v);
      else
        store_some(x, p.ldx - c, v);
    } else if (c + EACH <= p.ldx) {
      typedef __attribute__((ext_vector_type(EACH))) T V;
      typedef V Any __attribute__((aligned(sizeof(T))));
      *(Any*)x = V{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int k = 0; k < EACH; k++)
        if (c + k < p.ldx) x[k] = v[k];
    }
  }
}

}  // namespace ff
