// The plain products on the tiled kernel in fp16.
#include "tile_matmul.h"

namespace ff {

void backward_tiles_fp16(const Backward& b, hipStream_t st) {
  backward_tiles<_Float16>(b, st);
}

void split_tiles_fp16(const Matmul& q, Tile tile, hipStream_t st) {
  split_tiles<_Float16>(q, tile, st);
}

}  // namespace ff
