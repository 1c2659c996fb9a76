// Activations in 8 bits (the form is in feed_forward.h): pack and unpack.
//
// A thread holds eight neighbouring values, four threads a group of 32; the
// group's largest comes from two exchanges between neighbouring lanes.  One
// pass over the data, 16 + 8 bytes a thread: bound by memory.
#include "unpack8.h"

namespace ff {
namespace {

template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(const Pack p) {
  const long per = p.ldc / 8, total = p.m * per;  // per is a multiple of 4
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (long)gridDim.x * 256) {
    const long r = i / per, c = (i - r * per) * 8;
    float v[8];
    const T* x = (const T*)p.x + r * p.ldx + c;
    if (p.vec && c < p.n)
      load8(x, v);
    else
      load_some(x, p.n - c, v);
    // total is a multiple of 4: a group's four lanes are here together
    int e;
    *(uint2*)(p.codes + i * 8) = encode8<1, 2>(v, e);
    if ((i & 3) == 0) p.scales[i >> 2] = (unsigned char)(e + 127);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void unpack_kernel(const Pack p) {
  unpack_values<T>(p, (long)blockIdx.x * 256 + threadIdx.x,
                   (long)gridDim.x * 256);
}

}  // namespace

void launch_pack(const Pack& p, hipStream_t st) {
  const dim3 grid(rocps_grid_for(p.m * (p.ldc / 8), 256, 4096)), block(256);
  if (p.type == 0)
    hipLaunchKernelGGL((pack_kernel<__bf16>), grid, block, 0, st, p);
  else if (p.type == 1)
    hipLaunchKernelGGL((pack_kernel<_Float16>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL((pack_kernel<float>), grid, block, 0, st, p);
}

void launch_unpack(const Pack& p, hipStream_t st) {
  const int each = p.type == 2 ? 4 : 8;
  const dim3 grid(
      rocps_grid_for(p.m * ((p.ldx + each - 1) / each), 256, 4096));
  const dim3 block(256);
  if (p.type == 0)
    hipLaunchKernelGGL((unpack_kernel<__bf16>), grid, block, 0, st, p);
  else if (p.type == 1)
    hipLaunchKernelGGL((unpack_kernel<_Float16>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL((unpack_kernel<float>), grid, block, 0, st, p);
}

}  // namespace ff
