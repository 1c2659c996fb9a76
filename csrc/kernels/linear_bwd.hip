// Backward pass of the linear and the gated layer: the gradient of the
// pre-activations with its column sums, and the two products
//   dx = g W       dW = g^T x
// on the tiled product, with no transposed copies.
#include "feed_forward.h"
#include "linear.h"
#include "tile_gemm.h"

namespace ff {
namespace {

using tile::Operand;
using tile::Product;

// ---- the pre-activations' gradient ------------------------------------------
//
// A thread owns eight columns and walks down its run of rows; a block is 32
// threads wide and 8 rows high.  Each value is read once and written once:
// bound by memory.  The bias gradient's sums are taken from the fp32 values
// before they are rounded, over rows in a fixed order (no atomics): a run's
// sums go to `sums`, which a second kernel adds up.

// n valid values at p, zeros behind
template <typename T>
__device__ __forceinline__ void load_n(const T* p, long n, bool vec,
                                       float* v) {
  if (vec)
    load8(p, v);
  else
    load_some(p, n, v);
}

template <typename T, int ACT, bool GATED>
__global__ __launch_bounds__(256) void slope_kernel(const Slope s) {
  __shared__ float part[GATED ? 2 : 1][8][256];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long n = (long)blockIdx.x * 256 + tx * 8;
  const long run = (s.m + s.chunks - 1) / s.chunks;
  const long r0 = blockIdx.y * run;
  const long r1 = r0 + run < s.m ? r0 + run : s.m;
  const long left = s.n - n;
  float sum[8] = {}, sum2[8] = {};
  // columns behind n, up to the pitch's multiple of 8, are written as zeros
  if (left > 0) {
    for (long r = r0 + ty; r < r1; r += 8) {
      float d[8], g[8], u[8], o[8];
      load_n((const T*)s.dy + r * s.ldy + n, left, s.vec_dy, d);
      if constexpr (ACT != kNone) {
        const long at = r * s.ldp + n;
        if (s.codes != nullptr) {
          decode8(*(const uint2*)(s.codes + at), s.scales[at >> 5], g);
          if constexpr (GATED) {
            const long up = at + s.ldp / 2;
            decode8(*(const uint2*)(s.codes + up), s.scales[up >> 5], u);
          }
        } else {
          load8((const T*)s.pre + at, g);
          if constexpr (GATED) load8((const T*)s.pre + at + s.ldp / 2, u);
        }
      }
#pragma unroll
      for (int k = 0; k < 8; k++) {
        if constexpr (GATED) {
          const float da = d[k] * u[k] * slope<ACT>(g[k]);
          u[k] = d[k] * act<ACT>(g[k]);
          o[k] = da;
          if (k >= left) o[k] = u[k] = 0.f;
          sum2[k] += u[k];
        } else {
          o[k] = ACT == kNone ? d[k] : d[k] * slope<ACT>(g[k]);
          if (k >= left) o[k] = 0.f;
        }
        sum[k] += o[k];
      }
      if (s.out != nullptr) {
        T* out = (T*)s.out + r * s.ldo + n;
        if constexpr (GATED) {
          // the halves join at column n, wherever that is
          if (left >= 8 && (s.n & 7) == 0) {
            store8(out, o);
            store8(out + s.n, u);
          } else {
            store_some(out, left, o);
            store_some(out + s.n, left, u);
            if (left <= 8) {
#pragma unroll
              for (int k = 0; k < 8; k++)
                if (2 * s.n + k < s.ldo) out[2 * s.n - n + k] = (T)0.f;
            }
          }
        } else {
          store8(out, o);
        }
      }
    }
  }
  if (s.sums == nullptr) return;
#pragma unroll
  for (int k = 0; k < 8; k++) {
    part[0][ty][tx * 8 + k] = sum[k];
    if constexpr (GATED) part[1][ty][tx * 8 + k] = sum2[k];
  }
  __syncthreads();
  const long c = (long)blockIdx.x * 256 + threadIdx.x;
  if (c >= s.n) return;
  const long width = GATED ? 2 * s.n : s.n;
#pragma unroll
  for (int h = 0; h < (GATED ? 2 : 1); h++) {
    float t = 0.f;
#pragma unroll
    for (int y = 0; y < 8; y++) t += part[h][y][threadIdx.x];
    s.sums[blockIdx.y * width + h * s.n + c] = t;
  }
}

// sums over the runs: 64 columns a block, 4 threads a column
template <typename T>
__global__ __launch_bounds__(256) void sums_kernel(const float* sums,
                                                   int chunks, long width,
                                                   T* out) {
  __shared__ float part[4][64];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  const long c = (long)blockIdx.x * 64 + tx;
  float t = 0.f;
  if (c < width) {
#pragma unroll 8
    for (int r = ty; r < chunks; r += 4) t += sums[r * width + c];
  }
  part[ty][tx] = t;
  __syncthreads();
  if (ty == 0 && c < width)
    out[c] = (T)(part[0][tx] + part[1][tx] + part[2][tx] + part[3][tx]);
}

template <typename T, bool GATED>
void launch_slope_t(const Slope& s, hipStream_t st) {
  const dim3 grid((unsigned)((s.n + 255) / 256), s.chunks), block(256);
  if (s.act == kGelu)
    hipLaunchKernelGGL((slope_kernel<T, kGelu, GATED>), grid, block, 0, st, s);
  else if (s.act == kSilu)
    hipLaunchKernelGGL((slope_kernel<T, kSilu, GATED>), grid, block, 0, st, s);
  else if (s.act == kRelu)
    hipLaunchKernelGGL((slope_kernel<T, kRelu, GATED>), grid, block, 0, st, s);
  else if constexpr (!GATED)
    hipLaunchKernelGGL((slope_kernel<T, kNone, GATED>), grid, block, 0, st, s);
  if (s.sums != nullptr) {
    const long width = GATED ? 2 * s.n : s.n;
    hipLaunchKernelGGL((sums_kernel<T>), dim3((unsigned)((width + 63) / 64)),
                       block, 0, st, s.sums, s.chunks, width, (T*)s.dbias);
  }
}

// ---- the products -------------------------------------------------------------

template <typename T, int BM, int BN, bool AROWS, bool BROWS, bool SPLIT>
__global__ __launch_bounds__(256, BM == 256 ? 1 : 2)
void matmul_kernel(const Matmul q) {
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
    k0 = steps * split / q.splits * tile::BK;
    k1 = steps * (split + 1) / q.splits * tile::BK;
    if (k1 > q.k) k1 = q.k;
  }
  P prod;
  prod.run(smem, Operand{q.a, q.lda, q.m}, Operand{q.b, q.ldb, q.n}, m0, n0,
           k0, k1, 0);

  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, l = lane & 15;
#pragma unroll
  for (int p = 0; p < P::FN / 2; p++) {
    const long n = n0 + (wid & 1) * P::WN + p * 32 + g * 8;
#pragma unroll
    for (int i = 0; i < P::FM; i++) {
      const long m = m0 + (wid >> 1) * P::WM + i * 16 + l;
      if (m >= q.m || n >= q.n) continue;
      if constexpr (SPLIT) {
        float* o = q.part + ((long)split * q.m + m) * q.n + n;
        if (q.vec_out) {
          *(tile::f32x4*)o = prod.acc[i][2 * p];
          *(tile::f32x4*)(o + 4) = prod.acc[i][2 * p + 1];
        } else {
#pragma unroll
          for (int k = 0; k < 8; k++)
            if (n + k < q.n) o[k] = prod.acc[i][2 * p + (k >> 2)][k & 3];
        }
      } else {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = prod.acc[i][2 * p + (k >> 2)][k & 3];
        T* o = (T*)q.out + m * q.n + n;
        if (q.vec_out)
          store8(o, v);
        else
          store_some(o, q.n - n, v);
      }
    }
  }
}

// sums of the splits, in their order
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const float* part,
                                                   int splits, long count,
                                                   T* out, bool vec) {
  const long step = (long)gridDim.x * 256 * 8;
  for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * 8; i < count;
       i += step) {
    float v[8] = {};
    if (vec) {
      for (int s = 0; s < splits; s++) {
        const tile::f32x4* p = (const tile::f32x4*)(part + s * count + i);
        const tile::f32x4 a = p[0], b = p[1];
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] += a[k], v[4 + k] += b[k];
      }
      store8(out + i, v);
    } else {
      for (int s = 0; s < splits; s++)
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (i + k < count) v[k] += part[s * count + i + k];
      store_some(out + i, count - i, v);
    }
  }
}

template <typename T, int BM, int BN, bool AROWS, bool BROWS>
void launch_tiles(const Matmul& q, hipStream_t st) {
  const long tiles = ((q.m + BM - 1) / BM) * ((q.n + BN - 1) / BN);
  if (q.splits > 1) {
    hipLaunchKernelGGL((matmul_kernel<T, BM, BN, AROWS, BROWS, true>),
                       dim3((unsigned)(tiles * q.splits)), dim3(256), 0, st,
                       q);
    const long count = q.m * q.n;
    hipLaunchKernelGGL((join_kernel<T>), dim3(rocps_grid_for(count / 8, 256)),
                       dim3(256), 0, st, q.part, q.splits, count, (T*)q.out,
                       q.vec_out);
  } else {
    hipLaunchKernelGGL((matmul_kernel<T, BM, BN, AROWS, BROWS, false>),
                       dim3((unsigned)tiles), dim3(256), 0, st, q);
  }
}

bool big_tiles(long m, long n, long k) {
  return ((m + 255) / 256) * ((n + 255) / 256) >= 192;
}

template <typename T>
void launch_matmul_t(const Matmul& q, hipStream_t st) {
  const bool big = big_tiles(q.m, q.n, q.k);
  if (q.a_rows) {
    if (big) launch_tiles<T, 256, 256, true, true>(q, st);
    else launch_tiles<T, 128, 128, true, true>(q, st);
  } else {
    if (big) launch_tiles<T, 256, 256, false, true>(q, st);
    else launch_tiles<T, 128, 128, false, true>(q, st);
  }
}

__global__ __launch_bounds__(256) void repack_kernel(const short* x, long ldx,
                                                     long m, long n,
                                                     short* out, long ldo) {
  const long per = ldo / 8, total = m * per;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (long)gridDim.x * 256) {
    const long r = i / per, c = (i - r * per) * 8;
    tile::i16x8 v;
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = c + k < n ? x[r * ldx + c + k] : 0;
    *(tile::i16x8*)(out + r * ldo + c) = v;
  }
}

}  // namespace

int slope_chunks(long m, long n) {
  // some 1024 blocks, of 32 rows at least
  const long strips = (n + 255) / 256;
  long c = 1024 / strips;
  const long most = (m + 31) / 32;
  c = c < 1 ? 1 : (c > most ? most : c);
  return (int)(c > 256 ? 256 : c);
}

void launch_slope(const Slope& s, hipStream_t st) {
  if (s.type == 0) {
    if (s.gated) launch_slope_t<__bf16, true>(s, st);
    else launch_slope_t<__bf16, false>(s, st);
  } else {
    if (s.gated) launch_slope_t<_Float16, true>(s, st);
    else launch_slope_t<_Float16, false>(s, st);
  }
}

int matmul_splits(long m, long n, long k) {
  if (big_tiles(m, n, k)) return 1;
  const long tiles = ((m + 127) / 128) * ((n + 127) / 128);
  const long steps = (k + tile::BK - 1) / tile::BK;
  long s = 512 / tiles;               // two blocks on each of 256 CUs
  if (s > steps / 4) s = steps / 4;   // of four steps at least
  return (int)(s < 1 ? 1 : s);
}

void launch_matmul(const Matmul& q, hipStream_t st) {
  if (q.type == 0) launch_matmul_t<__bf16>(q, st);
  else launch_matmul_t<_Float16>(q, st);
}

void launch_repack(const void* x, long ldx, long m, long n, void* out,
                   long ldo, hipStream_t st) {
  hipLaunchKernelGGL(repack_kernel, dim3(rocps_grid_for(m * (ldo / 8), 256)),
                     dim3(256), 0, st, (const short*)x, ldx, m, n,
                     (short*)out, ldo);
}

}  // namespace ff
