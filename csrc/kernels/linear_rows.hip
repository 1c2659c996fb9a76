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
// to 64; its eight waves take the k's in turns of 64 and add their sums up
// through LDS.  No sums go through memory and there is one launch, so a single
// token costs what its weights do: 4096 -> 2 x 8192 takes 26.1 us (5.1 TB/s),
// what a large copy reaches.
//
// Each wave moves its share of both operands through LDS of its own, without
// barriers: eight rows of 128 bytes a load.  Read into registers as the matrix
// instruction wants them, a quarter of a wave touches 16 rows, and such loads
// pass at 16 bytes a clock: 24 rows of 4096 -> 4096 took 14.1 us so, of 4096 ->
// 16384 46.5, of 8192 -> 2048 22.5; these take 7.9, 33 and 9.9.
//
// Blocks begin at different k's: where rows are a power of two apart, they
// would all read from a few of the memory's channels at a time (4096 -> 2 x
// 8192: 29.3 us).
// (Rows of odd lengths are copied first: read as they lie, 16 bytes at any
// address, 24 rows of 4095 -> 4095 took 39 us, with the copy of the weights
// 34.)
//
// S turns are in flight.  Two are faster where one row's k is long and no more
// than one block comes to a CU (16 x 16384 -> 1024: 13.0 us, with one 15.3),
// and slower where their LDS keeps blocks from sharing it (16 x 1024 -> 32768:
// 20.4 and 16.5).
constexpr int kWaves = 8;

template <typename T, int MF, int S, bool GATED, int KEEP>
__global__ __launch_bounds__(64 * kWaves) void rows_kernel(const Forward f) {
  constexpr int H = GATED ? 2 : 1;
  constexpr int LOADS = 2 * (H + MF);  // a turn, 1 KB each
  constexpr int OWN = S * LOADS * 1024;  // a wave's part of LDS
  static_assert(OWN >= H * MF * 1024, "the sums too");
  __shared__ __attribute__((aligned(1024))) char smem[kWaves * OWN];
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, l = lane & 15;
  const long n0 = (long)blockIdx.x * 16;
  const int k = (int)f.k;

  // a load takes eight rows of 128 bytes, the 16 bytes' places permuted as in
  // the tiled product
  tile::lds_char* const own = (tile::lds_char*)smem + wid * OWN;
  const int chunk = ((lane & 7) ^ (lane >> 3)) * 8;
  unsigned woff[2], xoff[2 * MF];
  const long rows = f.n - n0;
#pragma unroll
  for (int p = 0; p < 2; p++) {
    const long n = p * 8 + (lane >> 3);
    woff[p] = (unsigned)(((n < rows ? n : rows - 1) * f.ldw + chunk) * 2) +
              tile::LEAD;
  }
#pragma unroll
  for (int p = 0; p < 2 * MF; p++) {
    const long m = p * 8 + (lane >> 3);
    xoff[p] = (unsigned)(((m < f.m ? m : f.m - 1) * f.ldx + chunk) * 2) +
              tile::LEAD;
  }
  tile::Descriptor dw[H];
#pragma unroll
  for (int h = 0; h < H; h++)
    dw[h] = tile::descriptor(
        (const char*)f.w + (h * f.n + n0) * f.ldw * 2,
        (int)((((rows < 16 ? rows : 16) - 1) * f.ldw + tile::whole(k)) * 2) +
            tile::LEAD);
  const tile::Descriptor dx = tile::descriptor(
      (const char*)f.x,
      (int)(((f.m - 1) * f.ldx + tile::whole(k)) * 2) + tile::LEAD);

  f32x4 acc[H][MF];
#pragma unroll
  for (int h = 0; h < H; h++)
#pragma unroll
    for (int i = 0; i < MF; i++) acc[h][i] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int turns = (k + kWaves * 64 - 1) / (kWaves * 64);
  int turn = (int)((blockIdx.x >> 3) % turns);  // the XCD's blocks differ
  int left = turns;
  // the next turn's loads; past the last, of nothing
  auto load = [&](int stage) {
    const int at = left > 0 ? turn * (kWaves * 64) + wid * 64 : k;
    const bool in = at + chunk < k;
    tile::lds_char* to = own + stage * LOADS * 1024;
#pragma unroll
    for (int p = 0; p < LOADS; p++) {
      tile::set_m0(to + p * 1024);
      const unsigned off = p < 2 * H ? woff[p & 1] : xoff[p - 2 * H];
      const unsigned o = in ? off : tile::PAST;
      asm volatile("s_nop 0");
      tile::load_lds(p < 2 * H ? dw[p / 2] : dx, o, at * 2, 0);
    }
    turn = turn + 1 < turns ? turn + 1 : 0;
    left--;
  };
#pragma unroll
  for (int s = 0; s < S; s++) load(s);
  for (int j = 0; j < turns; j += S) {
#pragma unroll
    for (int s = 0; s < S; s++) {
      tile::wait<(S - 1) * LOADS, false>();
      typedef __attribute__((address_space(3))) i16x8 lds_v8;
      i16x8 a[2][H], b[2][MF];
      tile::lds_char* from = own + s * LOADS * 1024 + l * 128;
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int c = ((e * 4 + g) ^ (l & 7)) << 4;
#pragma unroll
        for (int h = 0; h < H; h++)
          a[e][h] = *(lds_v8*)(from + h * 2048 + c);
#pragma unroll
        for (int i = 0; i < MF; i++)
          b[e][i] = *(lds_v8*)(from + (H + i) * 2048 + c);
      }
      tile::wait<63, true>();
      load(s);
#pragma unroll
      for (int e = 0; e < 2; e++)
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
          for (int i = 0; i < MF; i++)
            acc[h][i] = tile::mfma_value<T>(a[e][h], b[e][i], acc[h][i]);
    }
  }
  tile::wait<0, false>();  // no load may write LDS from here on
  typedef __attribute__((address_space(3))) f32x4 lds_f4;
  lds_f4* const part = (lds_f4*)(tile::lds_char*)smem;
  constexpr int NEXT = OWN / 16;  // from one wave's sums to the next one's
#pragma unroll
  for (int h = 0; h < H; h++)
#pragma unroll
    for (int i = 0; i < MF; i++)
      part[wid * NEXT + (h * MF + i) * 64 + lane] = acc[h][i];
  __syncthreads();

  // thread: row m, eight of the sixteen columns; column j of row m is value
  // j % 4 of lane 16 (j / 4) + m % 16
  const int t = threadIdx.x;
  if (t >= MF * 32) return;
  const int m = t >> 1, j = (t & 1) * 8;
  const long n = n0 + j;
  float v[8], u[8];
  widen(bias8<T>(f, n, 0), v);
  if constexpr (GATED) widen(bias8<T>(f, n, f.n), u);
  Vec8<T> r = {};
  if constexpr (!GATED) r = residual8<T>(f, m, n);
#pragma unroll
  for (int s = 0; s < kWaves; s++)
#pragma unroll
    for (int q = 0; q < 2; q++) {
      const int from =
          s * NEXT + (m >> 4) * 64 + (j / 4 + q) * 16 + (m & 15);
      const f32x4 p = part[from];
#pragma unroll
      for (int e = 0; e < 4; e++) v[q * 4 + e] += p[e];
      if constexpr (GATED) {
        const f32x4 o = part[from + MF * 64];
#pragma unroll
        for (int e = 0; e < 4; e++) u[q * 4 + e] += o[e];
      }
    }
  finish8<T, KEEP, -1, GATED, 1, 2>(f, m, n, m < f.m, v, u, r);
}

template <typename T, int MF, int S, bool GATED>
void launch_rows(const Forward& f, hipStream_t st) {
  const dim3 grid((unsigned)((f.n + 15) / 16)), block(64 * kWaves);
  if (f.pre != nullptr)
    hipLaunchKernelGGL((rows_kernel<T, MF, S, GATED, kPre>), grid, block, 0,
                       st, f);
  else
    hipLaunchKernelGGL((rows_kernel<T, MF, S, GATED, kNothing>), grid, block,
                       0, st, f);
}

template <typename T, bool GATED>
void rows_by_count(const Forward& f, hipStream_t st) {
  if (f.m <= 16) {
    if (!GATED && f.n <= 16 * kCUs) launch_rows<T, 1, 2, GATED>(f, st);
    else launch_rows<T, 1, 1, GATED>(f, st);
  } else if (f.m <= 32) {
    launch_rows<T, 2, 1, GATED>(f, st);
  } else if (f.m <= 48) {
    launch_rows<T, 3, 1, GATED>(f, st);
  } else {
    launch_rows<T, 4, 1, GATED>(f, st);
  }
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
    widen(bias8<T>(f, n, 0), v);
    if constexpr (GATED) widen(bias8<T>(f, n, f.n), u);
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

void choose_forward(Forward& f) {
  const long width = f.gated ? 2 * f.n : f.n;
  const bool eight = f.codes != nullptr;
  // in 8 bits a group of 32 columns would be two blocks'
  const bool few = f.m <= 64 && !eight;
  const double rows = few ? rows_cost(f.m, f.n, f.k, f.gated) : 0;
  const double read = 2e-6 * width * f.k / 5.1;
  f.by_rows = few && rows <= tiles_for_few(read);
  if (f.by_rows) return;
  f.choice = choose_tile(f.m, width, f.k, f.gated,
                         eight ? 2 : f.pre != nullptr ? 1 : 0);
  const double us = f.choice.us > read ? f.choice.us : read;
  f.by_rows = few && rows <= tiles_for_few(us);
}

void launch_linear_forward(const Forward& f, hipStream_t st) {
  const bool bf = f.type == 0;
  if (f.by_rows) {
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
