// Which tile and how many splits of k a product of the tiled kernel takes.
//
// Measured on an MI355X, bf16:
//   tile       blocks   us a step of 64 k's          us a 256 x 256 of
//              a CU     one block    each of all the output, with all
//                       alone        CU's at once    CUs at it
//   256 x 256    1        1.40         1.40            13
//   256 x 128    1        0.80         0.80            15
//   128 x 192    1        0.61         0.61            14
//   128 x 128    2        0.50         0.42             9
//    64 x 128    2        0.36         0.27            12
//    64 x  64    4        0.34         0.17             8
// and with pre-activations kept, 3 more where one block has the CU and 5 more
// where they share it; in 8 bits 9 and 8 more.
// A larger tile does more with what it reads; a smaller one leaves fewer CUs
// without work at the end, and two blocks on a CU write one's results while
// they multiply the other's.  The choice is the least time of the fullest CU.
// For 4096 x 4096 x 8192 (both operands by k) the tiles take 187, 214, 235,
// 222, 280 and 353 us, for 8192 x 768 x 4096 77, 51, 45, 55, 64 and 71, for
// 1024 x 1024 x 4096 78, 46, 39, 33, 28 and 26.
// Splits of k add partial sums in 32 bits, written, read and added up: their
// bytes at 4 TB/s and 4 us for the launch that joins them.
#pragma once

namespace ff {

enum Tile { k256x256, k256x128, k128x192, k128x128, k64x128, k64x64, kTiles };

struct TileChoice {
  Tile tile;
  int splits;
};

// `halves`: the gated layer's, whose tiles hold two runs of whole 32 columns.
// `keep`: what is kept, 0 nothing, 1 pre-activations, 2 those in 8 bits.
inline TileChoice choose_tile(long m, long n, long k, bool halves = false,
                              int keep = 0) {
  struct { long bm, bn; int per_cu; double alone, each, out; } const t[kTiles] =
      {{256, 256, 1, 1.40, 1.40, 13}, {256, 128, 1, 0.80, 0.80, 15},
       {128, 192, 1, 0.61, 0.61, 14}, {128, 128, 2, 0.50, 0.42, 9},
       {64, 128, 2, 0.36, 0.27, 12},  {64, 64, 4, 0.34, 0.17, 8}};
  const long cus = 256;
  const long steps = (k + 63) / 64;
  TileChoice best{k128x128, 1};
  double least = -1;
  for (int i = 0; i < kTiles; i++) {
    if (halves && (t[i].bn == 192 || t[i].bn == 64)) continue;
    const long tiles = ((m + t[i].bm - 1) / t[i].bm) *
                       ((n + t[i].bn - 1) / t[i].bn);
    const double more = keep == 0 ? 0
                        : t[i].per_cu == 1 ? (keep == 1 ? 3 : 9)
                                           : (keep == 1 ? 5 : 8);
    const double out = (t[i].out + more) * t[i].bm * t[i].bn / 65536;
    for (int s = 1; s <= 16 && (s == 1 || s * 4 <= steps); s++) {
      const long each = (tiles * s + cus - 1) / cus;  // of the fullest CU
      const long rest = each % t[i].per_cu;
      double last = 0;
      if (rest != 0)
        last = rest * t[i].each > t[i].alone ? rest * t[i].each : t[i].alone;
      double us = ((steps + s - 1) / s) * ((each - rest) * t[i].each + last);
      us += each * out;
      if (s > 1) us += 4 + s * 2e-6 * m * n;
      if (least < 0 || us < least) {
        least = us;
        best = {(Tile)i, s};
      }
      if (tiles * s >= 4 * cus) break;
    }
  }
  return best;
}

}  // namespace ff
