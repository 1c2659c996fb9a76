// Forward pass of the linear and the gated layer where the tiled product does
// not do it alone: few rows, which are bound by reading the weights once, and
// products whose k is split over blocks.
#include "forward_finish.h"
#include "tile_gemm.h"

namespace ff {
namespace {

using tile::f32x4;
using tile::i16x8;

// ---- few rows ---------------------------------------------------------------
//
// A block owns 16 rows of the weights (of each projection) and all of x's, up
// to 32; its eight waves take the k's in turns of 64 and add their sums up
// through LDS.  Weights go from memory to the matrix instruction's registers
// (lane l, 16 bytes: row l % 16, k's 8 (l / 16)..), each read by one wave
// alone, so there is nothing to stage; four turns are loaded before the first
// is used.  x comes from the L2.  No sums go through memory and there is one
// launch, so a single token costs what its weights do: 4096 -> 2 x 8192 takes
// 29.9 us (4.5 TB/s), 4096 -> 4096 8.1 us, 16 rows of that 10.8, 32 rows 13.8.
// From there on x's loads are more than the weights': 40 rows take 17.6 us,
// the tiled product with k split six times 14.9 (and 14.3 for 32).  Rows of odd
// lengths are copied first: read as they lie, 16 bytes at any address, 24 rows
// of 4095 -> 4095 take 39 us, with the copy of the weights 34.
constexpr int kWaves = 8, kTurns = 4;

template <typename T, int MF, bool GATED, int KEEP>
__global__ __launch_bounds__(64 * kWaves) void rows_kernel(const Forward f) {
  constexpr int H = GATED ? 2 : 1;
  __shared__ f32x4 part[kWaves][H][MF][64];
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, l = lane & 15;
  const long n0 = (long)blockIdx.x * 16;
  const long row = n0 + l < f.n ? n0 + l : f.n - 1;
  const T* w = (const T*)f.w + row * f.ldw + g * 8;
  const T* x[MF];
#pragma unroll
  for (int i = 0; i < MF; i++) {
    const long m = i * 16 + l < f.m ? i * 16 + l : f.m - 1;
    x[i] = (const T*)f.x + m * f.ldx + g * 8;
  }
  f32x4 acc[H][MF];
#pragma unroll
  for (int h = 0; h < H; h++)
#pragma unroll
    for (int i = 0; i < MF; i++) acc[h][i] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int k = (int)f.k;
  for (int k0 = wid * 64; k0 < k; k0 += kWaves * kTurns * 64) {
    i16x8 a[kTurns][2][H], b[kTurns][2][MF];
#pragma unroll
    for (int t = 0; t < kTurns; t++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int at = k0 + t * kWaves * 64 + e * 32;
        // rows end at whole 8's, with zeros behind k: all eight or none
        const bool in = at + g * 8 < k;
#pragma unroll
        for (int h = 0; h < H; h++)
          a[t][e][h] = in ? *(const i16x8*)(w + h * f.n * f.ldw + at)
                          : i16x8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < MF; i++)
          b[t][e][i] = in ? *(const i16x8*)(x[i] + at)
                          : i16x8{0, 0, 0, 0, 0, 0, 0, 0};
      }
#pragma unroll
    for (int t = 0; t < kTurns; t++)
#pragma unroll
      for (int e = 0; e < 2; e++)
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
          for (int i = 0; i < MF; i++)
            acc[h][i] = tile::mfma_value<T>(a[t][e][h], b[t][e][i], acc[h][i]);
  }
#pragma unroll
  for (int h = 0; h < H; h++)
#pragma unroll
    for (int i = 0; i < MF; i++) part[wid][h][i][lane] = acc[h][i];
  __syncthreads();

  // thread: row m, eight of the sixteen columns; column c of row m is value
  // c % 4 of lane 16 (c / 4) + m % 16
  const int t = threadIdx.x;
  if (t >= MF * 32) return;
  const int m = t >> 1, c = (t & 1) * 8;
  float v[8], u[8];
  bias8<T>(f, n0 + c, 0, v);
  if constexpr (GATED) bias8<T>(f, n0 + c, f.n, u);
  Vec8<T> r = {};
  if constexpr (!GATED) r = residual8<T>(f, m, n0 + c);
#pragma unroll
  for (int s = 0; s < kWaves; s++)
#pragma unroll
    for (int q = 0; q < 2; q++) {
      const int from = (c / 4 + q) * 16 + (m & 15);
      const f32x4 p = part[s][0][m >> 4][from];
#pragma unroll
      for (int r = 0; r < 4; r++) v[q * 4 + r] += p[r];
      if constexpr (GATED) {
        const f32x4 o = part[s][1][m >> 4][from];
#pragma unroll
        for (int r = 0; r < 4; r++) u[q * 4 + r] += o[r];
      }
    }
  finish8<T, KEEP, -1, GATED, 1, 2>(f, m, n0 + c, m < f.m, v, u, r);
}

template <typename T, int MF, bool GATED>
void launch_rows(const Forward& f, hipStream_t st) {
  const dim3 grid((unsigned)((f.n + 15) / 16)), block(64 * kWaves);
  if (f.pre != nullptr)
    hipLaunchKernelGGL((rows_kernel<T, MF, GATED, kPre>), grid, block, 0, st,
                       f);
  else
    hipLaunchKernelGGL((rows_kernel<T, MF, GATED, kNothing>), grid, block, 0,
                       st, f);
}

template <typename T, bool GATED>
void rows_by_count(const Forward& f, hipStream_t st) {
  if (f.m <= 16) launch_rows<T, 1, GATED>(f, st);
  else launch_rows<T, 2, GATED>(f, st);
}

// ---- splits of k ------------------------------------------------------------

// A thread takes eight columns of a row (and the same of the up half) of all
// splits, in their order; four threads hold a group of 32 columns.
template <typename T, bool GATED, int KEEP>
__global__ __launch_bounds__(256) void join_forward_kernel(const Forward f) {
  const long per = (f.n + 31) / 32 * 4, total = f.m * per;
  const long width = GATED ? 2 * f.n : f.n;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (long)gridDim.x * 256) {
    const long m = i / per, n = (i - m * per) * 8;
    float v[8], u[8];
    bias8<T>(f, n, 0, v);
    if constexpr (GATED) bias8<T>(f, n, f.n, u);
    Vec8<T> r = {};
    if constexpr (!GATED) r = residual8<T>(f, m, n);
    for (int s = 0; s < f.choice.splits; s++) {
      const float* p = f.part + ((long)s * f.m + m) * width + n;
      float a[8];
      load_some(p, f.n - n, a);
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] += a[k];
      if constexpr (GATED) {
        load_some(p + f.n, f.n - n, a);
#pragma unroll
        for (int k = 0; k < 8; k++) u[k] += a[k];
      }
    }
    finish8<T, KEEP, -1, GATED, 1, 2>(f, m, n, true, v, u, r);
  }
}

template <typename T, bool GATED>
void join_forward(const Forward& f, hipStream_t st) {
  const dim3 grid(rocps_grid_for(f.m * ((f.n + 31) / 32 * 4), 256, 4096));
  const dim3 block(256);
  if (f.codes != nullptr)
    hipLaunchKernelGGL((join_forward_kernel<T, GATED, k8>), grid, block, 0, st,
                       f);
  else if (f.pre != nullptr)
    hipLaunchKernelGGL((join_forward_kernel<T, GATED, kPre>), grid, block, 0,
                       st, f);
  else
    hipLaunchKernelGGL((join_forward_kernel<T, GATED, kNothing>), grid, block,
                       0, st, f);
}

}  // namespace

bool forward_by_rows(const Forward& f) {
  // a group of 32 columns would be two blocks'
  return f.m <= 32 && f.codes == nullptr;
}

TileChoice forward_choice(const Forward& f) {
  return choose_tile(f.m, f.gated ? 2 * f.n : f.n, f.k, f.gated,
                     f.codes != nullptr ? 2 : f.pre != nullptr ? 1 : 0);
}

void launch_linear_forward(const Forward& f, hipStream_t st) {
  const bool bf = f.type == 0;
  if (forward_by_rows(f)) {
    if (f.gated) {
      if (bf) rows_by_count<__bf16, true>(f, st);
      else rows_by_count<_Float16, true>(f, st);
    } else {
      if (bf) rows_by_count<__bf16, false>(f, st);
      else rows_by_count<_Float16, false>(f, st);
    }
    return;
  }
  if (f.choice.splits == 1) {
    if (bf) forward_tiles_bf16(f, st);
    else forward_tiles_fp16(f, st);
    return;
  }
  Matmul q{};
  q.m = f.m, q.n = f.gated ? 2 * f.n : f.n, q.k = f.k;
  q.vec_out = q.n % 8 == 0;
  q.a = f.x, q.lda = f.ldx;
  q.b = f.w, q.ldb = f.ldw;
  q.part = f.part;
  q.splits = f.choice.splits;
  if (bf) split_tiles_bf16(q, f.choice.tile, st);
  else split_tiles_fp16(q, f.choice.tile, st);
  if (f.gated) {
    if (bf) join_forward<__bf16, true>(f, st);
    else join_forward<_Float16, true>(f, st);
  } else {
    if (bf) join_forward<__bf16, false>(f, st);
    else join_forward<_Float16, false>(f, st);
  }
}

}  // namespace ff
