// Backward pass of the linear and the gated layer: the gradient of the
// pre-activations with its column sums, and what follows the two products
//   dx = g W       dW = g^T x
// (tile_matmul.h).
#include "tile_gemm.h"
#include "unpack8.h"

namespace ff {
namespace {

// ---- the pre-activations' gradient ------------------------------------------
//
// A thread owns eight columns and walks down its run of rows; a block is 32
// threads wide and 8 rows high.  Each value is read once and written once:
// bound by memory.  The bias gradient's sums are taken from the fp32 values
// before they are rounded, over rows in a fixed order (no atomics): a run's
// sums go to `sums`, which blocks of the products' launch add up.

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
  if ((int)blockIdx.x >= s.strips) {
    const long id = (long)(blockIdx.x - s.strips) * gridDim.y + blockIdx.y;
    unpack_values<T>(
        s.input, id * 256 + threadIdx.x,
        (long)(gridDim.x - s.strips) * gridDim.y * 256);
    return;
  }
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
          if constexpr (GATED) {
            const long up = at + s.ldp / 2;
            load24((const unsigned short*)s.pre + at, s.low + at, g);
            load24((const unsigned short*)s.pre + up, s.low + up, u);
          } else {
            load8((const T*)s.pre + at, g);
          }
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

template <typename T, bool GATED>
void launch_slope_t(Slope s, hipStream_t st) {
  // without `out` and `sums` there is nothing but the input to do
  s.strips = s.out == nullptr && s.sums == nullptr ? 0 : (s.n + 255) / 256;
  int more = 0;
  if (s.input.codes != nullptr) {
    // a block for some 4096 values
    const long blocks = (s.input.m * s.input.ldx + 4095) / 4096;
    more = (int)((blocks + s.chunks - 1) / s.chunks);
  }
  if (s.strips + more == 0) return;
  const dim3 grid(s.strips + more, s.chunks), block(256);
  if (s.act == kGelu)
    hipLaunchKernelGGL((slope_kernel<T, kGelu, GATED>), grid, block, 0, st, s);
  else if (s.act == kSilu)
    hipLaunchKernelGGL((slope_kernel<T, kSilu, GATED>), grid, block, 0, st, s);
  else if (s.act == kRelu)
    hipLaunchKernelGGL((slope_kernel<T, kRelu, GATED>), grid, block, 0, st, s);
  else if constexpr (!GATED)
    hipLaunchKernelGGL((slope_kernel<T, kNone, GATED>), grid, block, 0, st, s);
}

// ---- splits of k ------------------------------------------------------------

// One product's sums of its splits, in their order; blocks from `first` on
// take the other's.
struct Join {
  const float* part;
  void* out;
  long count;
  int splits, blocks;
};

template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const Join a,
                                                   const Join b) {
  const bool one = (int)blockIdx.x < a.blocks;
  const Join j = one ? a : b;
  const int id = one ? blockIdx.x : blockIdx.x - a.blocks;
  T* out = (T*)j.out;
  const long step = (long)j.blocks * 256 * 8;
  for (long i = ((long)id * 256 + threadIdx.x) * 8; i < j.count; i += step) {
    float v[8] = {};
    for (int s = 0; s < j.splits; s++) {
      float x[8];
      load_some(j.part + s * j.count + i, j.count - i, x);
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] += x[k];
    }
    store_some(out + i, j.count - i, v);
  }
}

Join join_of(const Matmul& q) {
  const long count = q.splits > 1 ? q.m * q.n : 0;
  return {q.part, q.out, count, q.splits,
          count == 0 ? 0 : rocps_grid_for((count + 7) / 8, 256)};
}

__global__ __launch_bounds__(256) void repack_kernel(const Repack a,
                                                     const Repack b) {
  const long first = a.m * (a.ldo / 8), all = first + b.m * (b.ldo / 8);
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < all;
       i += (long)gridDim.x * 256) {
    const bool one = i < first;
    const Repack p = one ? a : b;
    const long j = one ? i : i - first, per = p.ldo / 8;
    const long r = j / per, c = (j - r * per) * 8;
    *(Vec8<short>*)((short*)p.out + r * p.ldo + c) =
        some8((const short*)p.x + r * p.ldx + c, p.n - c);
  }
}

}  // namespace

int slope_chunks(long m, long n) {
  // Some 1024 blocks, and where there is not work for so many, of 8 rows, one
  // a thread: 1531 x 515 takes 5.8 us so and 10.6 with 32 rows, 512 x 768 4.2
  // and 6.1.
  const long strips = (n + 255) / 256;
  long c = 1024 / strips;
  const long most = (m + 7) / 8;
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

void launch_backward(const Backward& q, hipStream_t st) {
  if (q.type == 0) backward_tiles_bf16(q, st);
  else backward_tiles_fp16(q, st);
  const Join a = join_of(q.dx), b = join_of(q.dw);
  if (a.blocks + b.blocks == 0) return;
  const dim3 grid(a.blocks + b.blocks), block(256);
  if (q.type == 0)
    hipLaunchKernelGGL((join_kernel<__bf16>), grid, block, 0, st, a, b);
  else
    hipLaunchKernelGGL((join_kernel<_Float16>), grid, block, 0, st, a, b);
}

void launch_repack(const Repack& a, const Repack& b, hipStream_t st) {
  const long all = a.m * (a.ldo / 8) + b.m * (b.ldo / 8);
  if (all == 0) return;
  hipLaunchKernelGGL(repack_kernel, dim3(rocps_grid_for(all, 256)), dim3(256),
                     0, st, a, b);
}

}  // namespace ff
