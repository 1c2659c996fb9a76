// Forward pass of the linear and the gated layer on the tiled product:
// bias, activation, residual and the pre-activations that training keeps are
// written from the tile's registers.
#include "feed_forward.h"
#include "linear.h"
#include "tile_gemm.h"

namespace ff {
namespace {

using tile::Operand;
using tile::Product;

// eight columns' bias, zeros behind the last one
template <typename T>
__device__ __forceinline__ void bias8(const T* b, long n, long cols, bool vec,
                                      float* v) {
  if (b == nullptr || n >= cols) {
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = 0.f;
  } else if (vec) {
    load8(b + n, v);
  } else {
    load_some(b + n, cols - n, v);
  }
}

enum Keep { kNothing = 0, k16 = 1, k8 = 2 };

// keeps eight pre-activations of row m, columns n.. of f.n
template <typename T, int KEEP>
__device__ __forceinline__ void keep_pre(const Forward& f, long m, long n,
                                         long half, bool live, float* v) {
  if constexpr (KEEP == k16) {
    if (live && n < f.n) store8((T*)f.pre + m * f.ldp + half + n, v);
  } else if constexpr (KEEP == k8) {
    // the four lanes of one row, 16 apart, hold one group of 32
    float w[8], top = 0.f;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      w[k] = n + k < f.n ? v[k] : 0.f;
      const float u = __builtin_fabsf(w[k]);
      top = is_finite(w[k]) && u > top ? u : top;
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const int e = scale_exp(top);
    if (live && (n & ~31L) < f.n) {
      const long at = m * f.ldp + half + n;
      *(uint2*)(f.codes + at) = encode8(w, e);
      if ((n & 31) == 0) f.scales[at >> 5] = (unsigned char)(e + 127);
    }
  }
}

// Each i, p, k below is a compile-time constant after unrolling (the sums
// stay in registers), which is why the activation is a template argument:
// with all of them inside, the loops are too large to unroll.
template <typename T, int KEEP, int ACT, bool GATED, typename P>
__device__ __forceinline__ void finish(const P& prod, const Forward& f,
                                       long m0, long n0) {
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, l = lane & 15;
  const T* bias = (const T*)f.bias;
  T* y = (T*)f.y;
  constexpr int COLS = GATED ? P::WN / 2 : P::WN;
#pragma unroll
  for (int p = 0; p < COLS / 32; p++) {
    const long n = n0 + (wid & 1) * COLS + p * 32 + g * 8;
    float b[8], bu[8];
    bias8(bias, n, f.n, f.vec_out, b);
    if constexpr (GATED)
      bias8(bias == nullptr ? bias : bias + f.n, n, f.n, f.vec_out, bu);
#pragma unroll
    for (int i = 0; i < P::FM; i++) {
      const long m = m0 + (wid >> 1) * P::WM + i * 16 + l;
      const bool live = m < f.m;
      float v[8], u[8];
#pragma unroll
      for (int k = 0; k < 8; k++)
        v[k] = prod.acc[i][2 * p + (k >> 2)][k & 3] + b[k];
      keep_pre<T, KEEP>(f, m, n, 0, live, v);
      if constexpr (GATED) {
#pragma unroll
        for (int k = 0; k < 8; k++)
          u[k] = prod.acc[i][P::FN / 2 + 2 * p + (k >> 2)][k & 3] + bu[k];
        keep_pre<T, KEEP>(f, m, n, f.ldp / 2, live, u);
      }
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] = act<ACT>(v[k]);
      if constexpr (GATED) {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] *= u[k];
      }
      if (live && n < f.n) {
        if (!GATED && f.res != nullptr) {
          if (f.vec_out)
            load8((const T*)f.res + m * f.ldr + n, u);
          else
            load_some((const T*)f.res + m * f.ldr + n, f.n - n, u);
#pragma unroll
          for (int k = 0; k < 8; k++) v[k] += u[k];
        }
        if (f.vec_out)
          store8(y + m * f.n + n, v);
        else
          store_some(y + m * f.n + n, f.n - n, v);
      }
    }
  }
}

template <typename T, int BM, int BN, bool GATED, int KEEP>
__global__ __launch_bounds__(256, BM == 256 ? 1 : 2)
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

template <typename T, int BM, int BN, bool GATED>
void launch(const Forward& f, hipStream_t st) {
  constexpr int COLS = GATED ? BN / 2 : BN;
  const long tiles = ((f.m + BM - 1) / BM) * ((f.n + COLS - 1) / COLS);
  const dim3 grid((unsigned)tiles), block(256);
  if (f.codes != nullptr)
    hipLaunchKernelGGL((forward_kernel<T, BM, BN, GATED, k8>), grid, block, 0,
                       st, f);
  else if (f.pre != nullptr)
    hipLaunchKernelGGL((forward_kernel<T, BM, BN, GATED, k16>), grid, block,
                       0, st, f);
  else
    hipLaunchKernelGGL((forward_kernel<T, BM, BN, GATED, kNothing>), grid,
                       block, 0, st, f);
}

template <typename T, bool GATED>
void dispatch(const Forward& f, hipStream_t st) {
  const long cols = GATED ? 2 * f.n : f.n;
  const long big = ((f.m + 255) / 256) * ((cols + 255) / 256);
  if (big >= 192)
    launch<T, 256, 256, GATED>(f, st);
  else
    launch<T, 128, 128, GATED>(f, st);
}

}  // namespace

void launch_linear_forward(const Forward& f, hipStream_t st) {
  if (f.type == 0) {
    if (f.gated) dispatch<__bf16, true>(f, st);
    else dispatch<__bf16, false>(f, st);
  } else {
    if (f.gated) dispatch<_Float16, true>(f, st);
    else dispatch<_Float16, false>(f, st);
  }
}

}  // namespace ff
