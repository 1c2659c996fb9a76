// The plain products on the tiled kernel in bf16.
#include "tile_matmul.h"

namespace ff {

void backward_tiles_bf16(const Backward& b, hipStream_t st) {
  backward_tiles<__bf16>(b, st);
}

void split_tiles_bf16(const Matmul& q, Tile tile, hipStream_t st) {
  split_tiles<__bf16>(q, tile, st);
}

}  // namespace ff
