// !!! This is a file automatically generated by hipify!!!
#include "hip/hip_runtime.h"
// Plain products on the tiled kernel, with k split where there are few tiles;
// one type's kernels, for tile_matmul_bf16.hip and tile_matmul_fp16.hip.
#pragma once

#include "feed_forward.h"
#include "linear.h"
#include "tile_gemm.h"

namespace ff {

using tile::Operand;
using tile::Product;

template <typename T, int BM, int BN, int BLOCKS, bool AROWS, bool BROWS,
          bool SPLIT>
__global__ __launch_bounds__(256, BLOCKS) void matmul_kernel(const Matmul q) {
  using P = Product<T, BM, BN, AROWS, BROWS, false>;
  __shared__ __attribute__((aligned(1024))) char smem[P::LDS];
  const int mt = (int)((q.m + BM - 1) / BM), nt = (int)((q.n + BN - 1) / BN);
  const int tiles = mt * nt;
  int tm, tn, split = 0;
  if constexpr (SPLIT) {
    split = blockIdx.x / tiles;
    tile::tile_of(blockIdx.x % tiles, tiles, mt, nt, tm, tn);
  } else {
    tile::tile_of(blockIdx.x, tiles, mt, nt, tm, tn);
  }
  const long m0 = (long)tm * BM, n0 = (long)tn * BN;
  long k0 = 0, k1 = q.k;
  if constexpr (SPLIT) {  // runs of whole steps
    const long steps = (q.k + tile::BK - 1) / tile::BK;
    k0 = steps * split / q.choice.splits * tile::BK;
    k1 = steps * (split + 1) / q.choice.splits * tile::BK;
    if (k1 > q.k) k1 = q.k;
  }
  P prod;
  prod.run(smem, Operand{q.a, q.lda, q.m}, Operand{q.b, q.ldb, q.n}, m0, n0,
           k0, k1, 0);

  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int p = 0; p < P::FN / 2; p++) {
    const long n = n0 + (wid & 1) * P::WN + p * 32 + P::column(lane);
#pragma unroll
    for (int i = 0; i < P::FM; i++) {
      const long m = m0 + (wid >> 1) * P::WM + i * 16 + (lane & 15);
      float v[8];
      prod.eight(i, p, v);
      if (m >= q.m || n >= q.n) continue;
      if constexpr (SPLIT) {
        float* o = q.part + ((long)split * q.m + m) * q.n + n;
        if (q.vec_out) {
          *(tile::f32x4*)o = tile::f32x4{v[0], v[1], v[2], v[3]};
          *(tile::f32x4*)(o + 4) = tile::f32x4{v[4], v[5], v[6], v[7]};
        } else {
          store_some(o, q.n - n, v);
        }
      } else {
        T* o = (T*)q.out + m * q.n + n;
        if (q.vec_out)
          store8(o, v);
        else
          store_some(o, q.n - n, v);
      }
    }
  }
}

template <typename T, int BM, int BN, int BLOCKS, bool AROWS, bool BROWS,
          bool SPLIT>
void launch_tiles(const Matmul& q, hipStream_t st) {
  const long tiles = ((q.m + BM - 1) / BM) * ((q.n + BN - 1) / BN);
  const int splits = SPLIT ? q.choice.splits : 1;
  hipLaunchKernelGGL(
      (matmul_kernel<T, BM, BN, BLOCKS, AROWS, BROWS, SPLIT>),
      dim3((unsigned)(tiles * splits)), dim3(256), 0, st, q);
}

template <typename T, bool AROWS, bool BROWS, bool SPLIT>
void by_tile(const Matmul& q, hipStream_t st) {
  switch (q.choice.tile) {
    case k256x256:
      return launch_tiles<T, 256, 256, 1, AROWS, BROWS, SPLIT>(q, st);
    case k256x128:
      return launch_tiles<T, 256, 128, 1, AROWS, BROWS, SPLIT>(q, st);
    case k128x192:
      return launch_tiles<T, 128, 192, 1, AROWS, BROWS, SPLIT>(q, st);
    case k128x128:
      return launch_tiles<T, 128, 128, 2, AROWS, BROWS, SPLIT>(q, st);
    case k64x128:
      return launch_tiles<T, 64, 128, 2, AROWS, BROWS, SPLIT>(q, st);
    default:
      return launch_tiles<T, 64, 64, 4, AROWS, BROWS, SPLIT>(q, st);
  }
}

template <typename T>
void matmul_tiles(const Matmul& q, hipStream_t st) {
  if (q.choice.splits > 1) {
    if (q.a_rows) by_tile<T, true, true, true>(q, st);
    else by_tile<T, false, true, true>(q, st);
  } else {
    if (q.a_rows) by_tile<T, true, true, false>(q, st);
    else by_tile<T, false, true, false>(q, st);
  }
}

}  // namespace ff
