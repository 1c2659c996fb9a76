// The forward kernels of the linear and the gated layer in bf16.
#include "linear_fwd.h"

namespace ff {

void forward_tiles_bf16(const Forward& f, hipStream_t st) {
  forward_tiles<__bf16>(f, st);
}

}  // namespace ff
