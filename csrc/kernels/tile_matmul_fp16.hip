// The plain products on the tiled kernel in fp16.
#include "tile_matmul.h"

namespace ff {

void matmul_tiles_fp16(const Matmul& q, hipStream_t st) {
  matmul_tiles<_Float16>(q, st);
}

void split_tiles_fp16(const Matmul& q, hipStream_t st) {
  by_tile<_Float16, false, false, true>(q, st);
}

}  // namespace ff
