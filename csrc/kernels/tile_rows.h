// Results of the tiled product on their way to memory: whole rows of a wave's
// part, turned in LDS.
//
// A lane holds eight columns of one row, and the 16 lanes that a store passes
// at a time hold 16 different rows: 16 bytes a clock, a quarter of what
// neighbouring lanes with neighbouring columns reach.  So the 16 rows that a
// wave has of each block row go through LDS of its own, without barriers.  The
// forward pass of 4096 x 2048 -> 2 x 5632 in training takes 184 us so and 190
// straight from the lanes, that of 4096 x 2048 -> 5631 (with no row at whole
// 16 bytes) 97 and 103, the backward products of 8192 x 4096 -> 4096 460 and
// 476.
#pragma once

#include "tile_gemm.h"

namespace tile {

// COLS columns of BYTES bytes each, eight of them a lane's.
template <int COLS, int BYTES>
struct Turned {
  static constexpr int ROW = COLS * BYTES;    // bytes
  static constexpr int PITCH = ROW + 16;      // no two rows in the same banks
  static constexpr int LDS = 16 * PITCH;      // of a wave
  static constexpr int CHUNKS = ROW / 16;     // 16 bytes each
  static constexpr int READS = (CHUNKS + 3) / 4;
  static_assert(ROW % 16 == 0, "whole chunks");

  // lane's row and chunk of read r
  static __device__ __forceinline__ int row(int lane, int r) {
    return (r * 64 + lane) / CHUNKS;
  }
  static __device__ __forceinline__ int chunk(int lane, int r) {
    return (r * 64 + lane) % CHUNKS;
  }
  template <typename V>
  static __device__ __forceinline__ void put(lds_char* own, int row, int column,
                                             V v) {
    typedef __attribute__((address_space(3))) V lds_v;
    *(lds_v*)(own + row * PITCH + column * BYTES) = v;
  }
  template <typename V>
  static __device__ __forceinline__ V get(lds_char* own, int lane, int r) {
    typedef __attribute__((address_space(3))) V lds_v;
    static_assert(sizeof(V) == 16, "a chunk");
    return *(lds_v*)(own + row(lane, r) * PITCH + chunk(lane, r) * 16);
  }
};

}  // namespace tile
