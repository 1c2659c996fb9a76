// The plain products on the tiled kernel in bf16.
#include "tile_matmul.h"

namespace ff {

void matmul_tiles_bf16(const Matmul& q, hipStream_t st) {
  matmul_tiles<__bf16>(q, st);
}

void split_tiles_bf16(const Matmul& q, hipStream_t st) {
  by_tile<__bf16, false, false, true>(q, st);
}

}  // namespace ff
