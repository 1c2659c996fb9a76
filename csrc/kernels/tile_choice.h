// Which tile and how many splits of k a product of the tiled kernel takes.
//
// What a step of 64 k's and a tile's end cost, in us, bf16 on an MI355X:
//   tile       blocks   a step: one     each of all the CU's,    256 x 256 of
//              a CU     block alone     by k       by rows       the output
//   256 x 256    1        1.40          1.23         1.20        12.2
//   256 x 128    1        0.80          0.69         0.76        13.0
//   128 x 192    1        0.60          0.54         0.69        13.7
//   128 x 128    2        0.40          0.39         0.41         8.6
//    64 x 128    2        0.33          0.27         0.33        12.3
//    64 x  64    4        0.30          0.17         0.21         9.5
// and with pre-activations kept, 3 more where one block has the CU and 5 more
// where they share it; in 8 bits 9 and 8 more.  They are within a tenth or so
// of what single products take, and chosen so that the rules below choose
// well: over 82 shapes of the forward pass, each with pre-activations kept and
// not, and 83 of the backward pass, of 70 to 16384 rows and widths of 200 to
// 30528, each with every tile and up to eight splits measured, the choice is
// 1.9% and 1.3% slower than the best on average and 43% and 16% at most
// (profiles/feed_forward_tile_sweep.txt).
// A larger tile does more with what it reads; a smaller one leaves fewer CUs
// without work at the end, and two blocks on a CU write one's results while
// they multiply the other's.  The choice is the least time of the fullest CU.
// For 4096 x 4096 x 8192 (both operands by k) the tiles take 185, 213, 238,
// 223, 293 and 369 us, for 8192 x 768 x 4096 73, 51, 46, 52, 68 and 74, for
// 1024 x 1024 x 4096 71, 45, 38, 34, 30 and 28.
// Splits of k add partial sums in 32 bits, written, read and added up: 4.5 us
// for the launch that joins them, and their bytes.
#pragma once

namespace ff {

enum Tile { k256x256, k256x128, k128x192, k128x128, k64x128, k64x64, kTiles };

struct TileChoice {
  Tile tile;
  int splits;
  double us;
};

struct TileCost {
  long bm, bn;
  int per_cu;
  double alone, each, rows, out;
};

inline const TileCost& tile_cost(int t) {
  static const TileCost costs[kTiles] = {
      {256, 256, 1, 1.40, 1.23, 1.20, 12.2},
      {256, 128, 1, 0.80, 0.69, 0.76, 13.0},
      {128, 192, 1, 0.60, 0.54, 0.69, 13.7},
      {128, 128, 2, 0.40, 0.39, 0.41, 8.6},
      {64, 128, 2, 0.33, 0.27, 0.33, 12.3},
      {64, 64, 4, 0.30, 0.17, 0.21, 9.5}};
  return costs[t];
}

constexpr long kCUs = 256;
constexpr double kJoin = 4.5, kJoinEach = 1.3e-6;  // us, and for a value's sum

inline long tile_count(const TileCost& t, long m, long n) {
  return ((m + t.bm - 1) / t.bm) * ((n + t.bn - 1) / t.bn);
}

// One product.  `halves`: the gated layer's, whose tiles hold two runs of
// whole 32 columns; `keep`: what is kept, 0 nothing, 1 pre-activations, 2
// those in 8 bits.
inline TileChoice choose_tile(long m, long n, long k, bool halves, int keep) {
  const long steps = (k + 63) / 64;
  TileChoice best{k128x128, 1, 0};
  double least = -1;
  for (int i = 0; i < kTiles; i++) {
    const TileCost& t = tile_cost(i);
    if (halves && (t.bn == 192 || t.bn == 64)) continue;
    const long tiles = tile_count(t, m, n);
    const double more = keep == 0 ? 0
                        : t.per_cu == 1 ? (keep == 1 ? 3 : 9)
                                        : (keep == 1 ? 5 : 8);
    const double out = (t.out + more) * t.bm * t.bn / 65536;
    for (int s = 1; s <= 16 && (s == 1 || s * 4 <= steps); s++) {
      const long each = (tiles * s + kCUs - 1) / kCUs;  // of the fullest CU
      const long rest = each % t.per_cu;
      double last = 0;
      if (rest != 0) last = rest * t.each > t.alone ? rest * t.each : t.alone;
      double us = ((steps + s - 1) / s) * ((each - rest) * t.each + last);
      us += each * out;
      if (s > 1) us += kJoin + s * kJoinEach * m * n;
      if (least < 0 || us < least) {
        least = us;
        best = {(Tile)i, s, us};
      }
      if (tiles * s >= 4 * kCUs) break;
    }
  }
  return best;
}

// Up to 64 rows have a kernel that goes by 16 columns (linear_rows.hip).  What
// it takes, in us past the launch: a turn of its own and one of the rows for
// every k, times the blocks that a CU gets; blocks that share a CU wait for
// each other's loads.  Against the tiles, of which a few rows fill little and
// which start more slowly:
//                           16 rows        32            48
//   4096 -> 4096            7.6   13.7     8.0   14.6    8.9   15.4 us
//   8192 -> 2048            9.2   16.5     9.9   16.8    12.2  17.6
//   4096 -> 16384           26.6  37.2     33.7  37.8    40.8  38.8
//   1024 -> 32768           16.5  15.4     20.9  15.6    26.6  16.0
//   gated, 16384 -> 1024    31.3  23.8     38.7  24.6    45.1  25.4
// Over 20 shapes of both layers and 1 to 48 rows the choice is 1.7% slower
// than the better one on average, and 58% at most (1 row of 16384 -> 1024).
inline double rows_cost(long m, long n, long k, bool gated) {
  const int h = gated ? 2 : 1;
  const long runs = (m + 15) / 16;
  const double blocks = (double)n / 16 / kCUs;
  return blocks <= 1 ? 1e-3 * k * h * (0.6 + 0.25 * runs)
                     : 1e-3 * k * blocks * (1.3 * h + 0.5 * runs);
}

inline double tiles_for_few(double us) { return 1.2 * us + 2; }

// Two products of one launch, in tiles of one size, the longer ones first: a
// CU that is done with its share of one goes on with the other, so what
// counts is that all CUs end together.  A product of no rows is none.
struct PairChoice {
  Tile tile;
  int splits[2];
  bool second_first;
};

inline PairChoice choose_pair(const long m[2], const long n[2],
                              const long k[2]) {
  PairChoice best{k128x128, {1, 1}, false};
  double least = -1;
  const long steps[2] = {(k[0] + 63) / 64, (k[1] + 63) / 64};
  for (int i = 0; i < kTiles; i++) {
    const TileCost& t = tile_cost(i);
    const double out = t.out * t.bm * t.bn / 65536;
    const long tiles[2] = {tile_count(t, m[0], n[0]),
                           tile_count(t, m[1], n[1])};
    static const int kSplits[8] = {1, 2, 3, 4, 6, 8, 12, 16};
    for (int a = 0; a < 8; a++) {
      const int s0 = kSplits[a];
      if (a > 0 && (tiles[0] == 0 || s0 * 4 > steps[0] ||
                    tiles[0] * s0 >= 4 * kCUs))
        break;
      for (int b = 0; b < 8; b++) {
        const int s1 = kSplits[b];
        if (b > 0 && (tiles[1] == 0 || s1 * 4 > steps[1] ||
                      tiles[1] * s1 >= 4 * kCUs))
          break;
        // each block's time where every CU has its fill, and the longest's
        const double c0 = ((steps[0] + s0 - 1) / s0) * t.rows + out;
        const double c1 = ((steps[1] + s1 - 1) / s1) * t.rows + out;
        const bool swap = tiles[0] == 0 || (tiles[1] != 0 && c1 > c0);
        const double cl = swap ? c1 : c0, cs = swap ? c0 : c1;
        const long nl = swap ? tiles[1] * s1 : tiles[0] * s0;
        long ns = swap ? tiles[0] * s0 : tiles[1] * s1;
        // the longer ones leave two classes of CUs, which the shorter fill
        const long q = nl / kCUs, r = nl % kCUs;
        double hi = (q + (r > 0)) * cl, lo = q * cl;
        const long nhi = r > 0 ? r : kCUs, nlo = kCUs - nhi;
        double end = nl > 0 ? hi : 0;
        while (ns > 0) {
          if (nlo > 0 && lo <= hi) {
            lo += cs;
            ns -= nlo;
            end = lo > end ? lo : end;
          } else {
            hi += cs;
            ns -= nhi;
            end = hi > end ? hi : end;
          }
        }
        const long most = (swap ? steps[1] + s1 - 1 : steps[0] + s0 - 1) /
                          (swap ? s1 : s0);
        // where CUs are shared, the longest block has most of one to itself
        const long total = tiles[0] * s0 + tiles[1] * s1;
        long share = (total + kCUs - 1) / kCUs;
        share = share < t.per_cu ? share : t.per_cu;
        const double with = t.rows * (1 + 0.5 * (share - 1));
        const double lone = most * (with > t.alone ? with : t.alone) + out;
        double us = end > lone ? end : lone;
        if (s0 > 1 || s1 > 1) us += kJoin;
        if (s0 > 1) us += s0 * kJoinEach * m[0] * n[0];
        if (s1 > 1) us += s1 * kJoinEach * m[1] * n[1];
        if (least < 0 || us < least) {
          least = us;
          best = {(Tile)i, {s0, s1}, swap};
        }
      }
    }
  }
  return best;
}

}  // namespace ff
