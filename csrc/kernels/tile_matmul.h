// Plain products on the tiled kernel: the backward pass's two in one launch,
// and the forward pass's with k split; one type's kernels, for
// tile_matmul_bf16.hip and tile_matmul_fp16.hip.
#pragma once

#include "feed_forward.h"
#include "linear.h"
#include "tile_gemm.h"
#include "tile_rows.h"

namespace ff {

using tile::Operand;
using tile::Product;

// 256 rows of the longest pitch end before the offset that loads nothing.
static_assert(256 * (kMaxPitch - 8) * 2 + tile::LEAD < tile::PAST,
              "a tile's extent");

// A wave's part of a tile, rows from m0 and columns from n0 on, to out[m][n].
template <typename P, typename O>
__device__ __forceinline__ void write_tile(const P& prod, char* smem, int wid,
                                           int lane, O* out, long m0, long n0,
                                           long m, long n) {
  using Turn = tile::Turned<P::WN, sizeof(O)>;
  static_assert(4 * Turn::LDS <= P::LDS, "the waves' rows");
  constexpr int EACH = 16 / sizeof(O);  // columns a chunk
  using V = __attribute__((ext_vector_type(EACH))) O;
  tile::lds_char* const own = (tile::lds_char*)smem + wid * Turn::LDS;
#pragma unroll
  for (int i = 0; i < P::FM; i++) {
#pragma unroll
    for (int p = 0; p < P::FN / 2; p++) {
      float v[8];
      prod.eight(i, p, v);
      const int c = p * 32 + P::column(lane);
      V u[8 / EACH];
#pragma unroll
      for (int k = 0; k < 8; k++) u[k / EACH][k % EACH] = (O)v[k];
#pragma unroll
      for (int k = 0; k < 8 / EACH; k++)
        Turn::put(own, lane & 15, c + k * EACH, u[k]);
    }
#pragma unroll
    for (int r = 0; r < Turn::READS; r++) {
      const V u = Turn::template get<V>(own, lane, r);
      const long row = m0 + i * 16 + Turn::row(lane, r);
      const long c = n0 + Turn::chunk(lane, r) * EACH;
      if (row < m && c < n) {
        O* to = out + row * n + c;
        if (c + EACH <= n) {
          typedef V Any __attribute__((aligned(sizeof(O))));
          *(Any*)to = u;
        } else {
#pragma unroll
          for (int k = 0; k < EACH; k++)
            if (c + k < n) to[k] = u[k];
        }
      }
    }
  }
}

// Block `id` of a product's tiles and splits.
template <typename T, int BM, int BN, bool AROWS, bool BROWS>
__device__ __forceinline__ void matmul_block(char* smem, const Matmul& q,
                                             int id) {
  using P = Product<T, BM, BN, AROWS, BROWS, false>;
  const int mt = (int)((q.m + BM - 1) / BM), nt = (int)((q.n + BN - 1) / BN);
  const int tiles = mt * nt;
  if (id >= tiles * q.splits) return;
  const int split = id / tiles;
  int tm, tn;
  tile::tile_of(id - split * tiles, tiles, mt, nt, tm, tn);
  const long m0 = (long)tm * BM, n0 = (long)tn * BN;
  // runs of whole steps
  const long steps = (q.k + tile::BK - 1) / tile::BK;
  const long k0 = steps * split / q.splits * tile::BK;
  long k1 = steps * (split + 1) / q.splits * tile::BK;
  if (k1 > q.k) k1 = q.k;
  P prod;
  prod.run(smem, Operand{q.a, q.lda, q.m}, Operand{q.b, q.ldb, q.n}, m0, n0,
           k0, k1, 0);

  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long mw = m0 + (wid >> 1) * P::WM, nw = n0 + (wid & 1) * P::WN;
  tile::barrier();  // the tiles' last reads are done
  if (q.splits == 1)
    write_tile<P>(prod, smem, wid, lane, (T*)q.out, mw, nw, q.m, q.n);
  else
    write_tile<P>(prod, smem, wid, lane, q.part + (long)split * q.m * q.n, mw,
                  nw, q.m, q.n);
}

template <typename T, int BM, int BN, int BLOCKS>
__global__ __launch_bounds__(256, BLOCKS) void split_kernel(const Matmul q) {
  __shared__ __attribute__((aligned(1024))) char
      smem[Product<T, BM, BN, false, false, false>::LDS];
  matmul_block<T, BM, BN, false, false>(smem, q, blockIdx.x);
}

// The bias gradient: 64 columns' sums over the runs, 4 threads a column.
template <typename T>
__device__ __forceinline__ void sum_block(char* smem, const Backward& b,
                                          int id) {
  float(*part)[64] = (float(*)[64])smem;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  const long c = (long)id * 64 + tx;
  float t = 0.f;
  if (c < b.width) {
#pragma unroll 8
    for (int r = ty; r < b.chunks; r += 4) t += b.sums[r * b.width + c];
  }
  part[ty][tx] = t;
  __syncthreads();
  if (ty == 0 && c < b.width)
    ((T*)b.dbias)[c] =
        (T)(part[0][tx] + part[1][tx] + part[2][tx] + part[3][tx]);
}

// Blocks: the longer product's, the other's, the sums'.  Each product's
// begin at a multiple of 8, so that their numbers say the XCD.
template <typename T, int BM, int BN, int BLOCKS>
__global__ __launch_bounds__(256, BLOCKS)
void backward_kernel(const Backward b, int first, int second) {
  constexpr int LDS = Product<T, BM, BN, true, true, false>::LDS;
  static_assert(LDS == Product<T, BM, BN, false, true, false>::LDS, "one");
  __shared__ __attribute__((aligned(1024))) char smem[LDS];
  const int id = blockIdx.x;
  if (id >= first + second)
    sum_block<T>(smem, b, id - first - second);
  else if ((id < first) == b.choice.second_first)
    matmul_block<T, BM, BN, true, true>(smem, b.dw,
                                        id < first ? id : id - first);
  else
    matmul_block<T, BM, BN, false, true>(smem, b.dx,
                                         id < first ? id : id - first);
}

template <typename T, int BM, int BN, int BLOCKS>
void launch_split(const Matmul& q, hipStream_t st) {
  const long tiles = ((q.m + BM - 1) / BM) * ((q.n + BN - 1) / BN);
  hipLaunchKernelGGL((split_kernel<T, BM, BN, BLOCKS>),
                     dim3((unsigned)(tiles * q.splits)), dim3(256), 0, st, q);
}

template <typename T, int BM, int BN, int BLOCKS>
void launch_pair(const Backward& b, hipStream_t st) {
  auto blocks = [](const Matmul& q) {
    const long tiles = ((q.m + BM - 1) / BM) * ((q.n + BN - 1) / BN);
    return (int)((tiles * q.splits + 7) / 8 * 8);
  };
  const int dx = blocks(b.dx), dw = blocks(b.dw);
  const int first = b.choice.second_first ? dw : dx;
  const int sums = b.sums == nullptr ? 0 : (int)((b.width + 63) / 64);
  hipLaunchKernelGGL((backward_kernel<T, BM, BN, BLOCKS>),
                     dim3((unsigned)(dx + dw + sums)), dim3(256), 0, st, b,
                     first, dx + dw - first);
}

template <typename T>
void split_tiles(const Matmul& q, Tile tile, hipStream_t st) {
  switch (tile) {
    case k256x256: return launch_split<T, 256, 256, 1>(q, st);
    case k256x128: return launch_split<T, 256, 128, 1>(q, st);
    case k128x192: return launch_split<T, 128, 192, 1>(q, st);
    case k128x128: return launch_split<T, 128, 128, 2>(q, st);
    case k64x128: return launch_split<T, 64, 128, 2>(q, st);
    default: return launch_split<T, 64, 64, 4>(q, st);
  }
}

template <typename T>
void backward_tiles(const Backward& b, hipStream_t st) {
  switch (b.choice.tile) {
    case k256x256: return launch_pair<T, 256, 256, 1>(b, st);
    case k256x128: return launch_pair<T, 256, 128, 1>(b, st);
    case k128x192: return launch_pair<T, 128, 192, 1>(b, st);
    case k128x128: return launch_pair<T, 128, 128, 2>(b, st);
    case k64x128: return launch_pair<T, 64, 128, 2>(b, st);
    default: return launch_pair<T, 64, 64, 4>(b, st);
  }
}

}  // namespace ff
