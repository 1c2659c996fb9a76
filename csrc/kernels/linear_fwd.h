// Forward pass of the linear and the gated layer on the tiled product; one
// type's kernels, for linear_fwd_bf16.hip and linear_fwd_fp16.hip.
#pragma once

#include "forward_finish.h"
#include "tile_gemm.h"

namespace ff {

using tile::Operand;
using tile::Product;

// Each i, p, k below is a compile-time constant after unrolling (the sums
// stay in registers), which is why the activation is a template argument:
// with all of them inside, the loops are too large to unroll.
template <typename T, int KEEP, int ACT, bool GATED, typename P>
__device__ __forceinline__ void finish(const P& prod, const Forward& f,
                                       long m0, long n0) {
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int COLS = GATED ? P::WN / 2 : P::WN;
  // The whole residual before the first store, which the compiler has to take
  // for one to the same place: one wait instead of one a row.  Its registers
  // are the fragments'.  Before the products, with their first loads, it costs
  // as much: 8192 x 768 -> 768 takes 18.0 us so and 16.9 here.
  constexpr int PAIRS = COLS / 32;
  Vec8<T> r[GATED ? 1 : PAIRS][P::FM] = {};
  if constexpr (!GATED) {
#pragma unroll
    for (int p = 0; p < PAIRS; p++)
#pragma unroll
      for (int i = 0; i < P::FM; i++)
        r[p][i] = residual8<T>(
            f, m0 + (wid >> 1) * P::WM + i * 16 + (lane & 15),
            n0 + (wid & 1) * COLS + p * 32 + P::column(lane));
  }
#pragma unroll
  for (int p = 0; p < PAIRS; p++) {
    const long n = n0 + (wid & 1) * COLS + p * 32 + P::column(lane);
    float b[8], bu[8];
    bias8<T>(f, n, 0, b);
    if constexpr (GATED) bias8<T>(f, n, f.n, bu);
#pragma unroll
    for (int i = 0; i < P::FM; i++) {
      const long m = m0 + (wid >> 1) * P::WM + i * 16 + (lane & 15);
      float v[8], u[8];
      prod.eight(i, p, v);
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] += b[k];
      if constexpr (GATED) {
        prod.eight(i, P::FN / 4 + p, u);
#pragma unroll
        for (int k = 0; k < 8; k++) u[k] += bu[k];
      }
      finish8<T, KEEP, ACT, GATED, 16, 32>(f, m, n, m < f.m, v, u,
                                           r[GATED ? 0 : p][i]);
    }
  }
}

template <typename T, int BM, int BN, int BLOCKS, bool GATED, int KEEP>
__global__ __launch_bounds__(256, BLOCKS)
void forward_kernel(const Forward f) {
  using P = Product<T, BM, BN, false, false, GATED>;
  __shared__ __attribute__((aligned(1024))) char smem[P::LDS];
  constexpr int COLS = GATED ? BN / 2 : BN;  // output columns of a tile
  const int mt = (int)((f.m + BM - 1) / BM);
  const int nt = (int)((f.n + COLS - 1) / COLS);
  int tm, tn;
  tile::tile_of(blockIdx.x, gridDim.x, mt, nt, tm, tn);
  const long m0 = (long)tm * BM, n0 = (long)tn * COLS;

  P prod;
  prod.run(smem, Operand{f.x, f.ldx, f.m}, Operand{f.w, f.ldw, f.n}, m0, n0,
           0, f.k, f.n);

  if (f.act == kGelu)
    finish<T, KEEP, kGelu, GATED>(prod, f, m0, n0);
  else if (f.act == kSilu)
    finish<T, KEEP, kSilu, GATED>(prod, f, m0, n0);
  else if (f.act == kRelu)
    finish<T, KEEP, kRelu, GATED>(prod, f, m0, n0);
  else if constexpr (!GATED && KEEP == kNothing)  // nothing to keep here
    finish<T, KEEP, kNone, GATED>(prod, f, m0, n0);
}

template <typename T, int BM, int BN, int BLOCKS, bool GATED>
void launch_forward(const Forward& f, hipStream_t st) {
  constexpr int COLS = GATED ? BN / 2 : BN;
  const long tiles = ((f.m + BM - 1) / BM) * ((f.n + COLS - 1) / COLS);
  const dim3 grid((unsigned)tiles), block(256);
  if (f.codes != nullptr)
    hipLaunchKernelGGL((forward_kernel<T, BM, BN, BLOCKS, GATED, k8>), grid,
                       block, 0, st, f);
  else if (f.pre != nullptr)
    hipLaunchKernelGGL((forward_kernel<T, BM, BN, BLOCKS, GATED, kPre>), grid,
                       block, 0, st, f);
  else
    hipLaunchKernelGGL((forward_kernel<T, BM, BN, BLOCKS, GATED, kNothing>),
                       grid, block, 0, st, f);
}

template <typename T>
void forward_tiles(const Forward& f, hipStream_t st) {
  if (f.gated) {
    switch (f.choice.tile) {
      case k256x256: return launch_forward<T, 256, 256, 1, true>(f, st);
      case k256x128: return launch_forward<T, 256, 128, 1, true>(f, st);
      case k128x128: return launch_forward<T, 128, 128, 2, true>(f, st);
      default: return launch_forward<T, 64, 128, 2, true>(f, st);
    }
  }
  switch (f.choice.tile) {
    case k256x256: return launch_forward<T, 256, 256, 1, false>(f, st);
    case k256x128: return launch_forward<T, 256, 128, 1, false>(f, st);
    case k128x192: return launch_forward<T, 128, 192, 1, false>(f, st);
    case k128x128: return launch_forward<T, 128, 128, 2, false>(f, st);
    case k64x128: return launch_forward<T, 64, 128, 2, false>(f, st);
    default: return launch_forward<T, 64, 64, 4, false>(f, st);
  }
}

}  // namespace ff
