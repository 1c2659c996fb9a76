// The forward kernels of the linear and the gated layer in fp16.
#include "linear_fwd.h"

namespace ff {

void forward_tiles_fp16(const Forward& f, hipStream_t st) {
  forward_tiles<_Float16>(f, st);
}

}  // namespace ff
