// Forward pass of the linear and the gated layer on the tiled product; one
// type's kernels, for linear_fwd_bf16.hip and linear_fwd_fp16.hip.
#pragma once

#include "forward_finish.h"
#include "tile_gemm.h"
#include "tile_rows.h"

namespace ff {

using tile::Operand;
using tile::Product;

// A wave's part of LDS after the products: 16 rows of each result.
template <int COLS, bool GATED, int KEEP>
struct Rows {
  using Wide = tile::Turned<COLS, 2>;    // 16-bit values
  using Narrow = tile::Turned<COLS, 1>;  // bytes
  static constexpr int H = GATED ? 2 : 1;
  static constexpr int PRE = Wide::LDS;  // behind y's: pre-activations
  static constexpr int LOW = PRE + (KEEP == kPre ? H * Wide::LDS : 0);
  static constexpr int LDS =
      LOW + (KEEP == k8 || (GATED && KEEP == kPre) ? H * Narrow::LDS : 0);
};

// Rows of bytes, 16 a lane, `limit` of them (whole eights) in a row; base: the
// first row's.
template <typename R>
__device__ __forceinline__ void store_bytes(tile::lds_char* own, int lane,
                                            unsigned char* base, long ldp,
                                            long m, long rows, long n,
                                            long limit) {
  using V = __attribute__((ext_vector_type(4))) unsigned;
  typedef V Any __attribute__((aligned(8)));
#pragma unroll
  for (int r = 0; r < R::READS; r++) {
    // the last read may be more than there is
    if (R::CHUNKS * 16 % 64 != 0 && r * 64 + lane >= R::CHUNKS * 16) break;
    const V v = R::template get<V>(own, lane, r);
    const long row = m + R::row(lane, r), c = n + R::chunk(lane, r) * 16;
    if (row >= rows || c >= limit) continue;
    unsigned char* to = base + row * ldp + c;
    if (c + 16 <= limit)
      *(Any*)to = v;
    else
      *(uint2*)to = make_uint2(v[0], v[1]);
  }
}

// Each i, p, k below is a compile-time constant after unrolling (the sums
// stay in registers), which is why the activation is a template argument:
// with all of them inside, the loops are too large to unroll.
template <typename T, int KEEP, int ACT, bool GATED, typename P>
__device__ __forceinline__ void finish(const P& prod, const Forward& f,
                                       char* smem, long m0, long n0) {
  constexpr int COLS = GATED ? P::WN / 2 : P::WN, PAIRS = COLS / 32;
  constexpr int H = GATED ? 2 : 1;
  using L = Rows<COLS, GATED, KEEP>;
  using Wide = typename L::Wide;
  using Narrow = typename L::Narrow;
  static_assert(4 * L::LDS <= P::LDS, "the waves' rows");
  static_assert(Wide::CHUNKS % 4 == 0, "whole reads");
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = lane & 15;
  tile::lds_char* const own = (tile::lds_char*)smem + wid * L::LDS;
  const long mw = m0 + (wid >> 1) * P::WM, nw = n0 + (wid & 1) * COLS;
  tile::barrier();  // the tiles' last reads are done

  // The whole residual before the first store, which the compiler has to take
  // for one to the same place: one wait instead of one a row.  Its registers
  // are the fragments'.  (Before the products, with their first loads, it is no
  // faster: 8192 x 768 -> 768 took 18.0 us so and 16.9 here.)
  Vec8<T> res[GATED ? 1 : P::FM][Wide::READS];
  if constexpr (!GATED) {
    if (f.res != nullptr) {
#pragma unroll
      for (int i = 0; i < P::FM; i++)
#pragma unroll
        for (int r = 0; r < Wide::READS; r++)
          res[i][r] = residual8<T>(f, mw + i * 16 + Wide::row(lane, r),
                                   nw + Wide::chunk(lane, r) * 8);
    }
  }
  Vec8<T> bias[H][PAIRS];
#pragma unroll
  for (int h = 0; h < H; h++)
#pragma unroll
    for (int p = 0; p < PAIRS; p++)
      bias[h][p] = bias8<T>(f, nw + p * 32 + P::column(lane), h * f.n);

#pragma unroll
  for (int i = 0; i < P::FM; i++) {
    const long m = mw + i * 16;
    if constexpr (!GATED) {
      if (f.res != nullptr) {
#pragma unroll
        for (int r = 0; r < Wide::READS; r++)
          Wide::put(own, Wide::row(lane, r), Wide::chunk(lane, r) * 8,
                    res[i][r]);
      }
    }
#pragma unroll
    for (int p = 0; p < PAIRS; p++) {
      const int c = p * 32 + P::column(lane);
      float v[H][8];
#pragma unroll
      for (int h = 0; h < H; h++) {
        prod.eight(i, h * (P::FN / 4) + p, v[h]);
#pragma unroll
        for (int k = 0; k < 8; k++) v[h][k] += (float)bias[h][p][k];
        if constexpr (KEEP == kPre) {
          tile::lds_char* const to = own + L::PRE + h * Wide::LDS;
          if constexpr (GATED) {
            u16x8 hi;
            const uint2 lo = split24(v[h], hi);
            Wide::put(to, l, c, hi);
            Narrow::put(own + L::LOW + h * Narrow::LDS, l, c,
                        u32x2{lo.x, lo.y});
          } else {
            Wide::put(to, l, c, to8<T>(v[h]));
          }
        } else if constexpr (KEEP == k8) {
          int e;
          const uint2 codes = codes8<16, 32>(f, nw + c, v[h], e);
          Narrow::put(own + L::LOW + h * Narrow::LDS, l, c,
                      u32x2{codes.x, codes.y});
          if (c % 32 == 0 && m + l < f.m && nw + c < f.n)
            f.scales[((m + l) * f.ldp + h * (f.ldp / 2) + nw + c) >> 5] =
                (unsigned char)(e + 127);
        }
      }
      act8<ACT>(v[0], ACT);
      if constexpr (GATED) {
#pragma unroll
        for (int k = 0; k < 8; k++) v[0][k] *= v[H - 1][k];
      } else if (f.res != nullptr) {
        typedef __attribute__((address_space(3))) Vec8<T> lds_v;
        const Vec8<T> r = *(lds_v*)(own + l * Wide::PITCH + c * 2);
#pragma unroll
        for (int k = 0; k < 8; k++) v[0][k] += (float)r[k];
      }
      Wide::put(own, l, c, to8<T>(v[0]));
    }
#pragma unroll
    for (int r = 0; r < Wide::READS; r++) {
      const long row = m + Wide::row(lane, r);
      const long n = nw + Wide::chunk(lane, r) * 8;
      const Vec8<T> y = Wide::template get<Vec8<T>>(own, lane, r);
      if (row < f.m && n < f.n) {
        put_some((T*)f.y + row * f.n + n, f.n - n, y);
        if constexpr (KEEP == kPre) {
#pragma unroll
          for (int h = 0; h < H; h++)
            *(Vec8<T>*)((T*)f.pre + row * f.ldp + h * (f.ldp / 2) + n) =
                Wide::template get<Vec8<T>>(own + L::PRE + h * Wide::LDS, lane,
                                            r);
        }
      }
    }
    if constexpr (KEEP == k8 || (GATED && KEEP == kPre)) {
      const long step = KEEP == k8 ? 32 : 8;
#pragma unroll
      for (int h = 0; h < H; h++)
        store_bytes<Narrow>(own + L::LOW + h * Narrow::LDS, lane,
                            (KEEP == k8 ? f.codes : f.low) + h * (f.ldp / 2),
                            f.ldp, m, f.m, nw, (f.n + step - 1) / step * step);
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
    finish<T, KEEP, kGelu, GATED>(prod, f, smem, m0, n0);
  else if (f.act == kSilu)
    finish<T, KEEP, kSilu, GATED>(prod, f, smem, m0, n0);
  else if (f.act == kRelu)
    finish<T, KEEP, kRelu, GATED>(prod, f, smem, m0, n0);
  else if constexpr (!GATED && KEEP == kNothing)  // nothing to keep here
    finish<T, KEEP, kNone, GATED>(prod, f, smem, m0, n0);
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
