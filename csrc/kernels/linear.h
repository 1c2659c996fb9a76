// Launchers of the linear and the gated layer and of activations in 8 bits.
// Types: 0 bf16, 1 fp16.  Activations: 0 none, 1 relu, 2 gelu (tanh), 3 silu.
#pragma once

#include <hip/hip_runtime.h>

#include "tile_choice.h"

namespace ff {

// Pitches of operands of the tiled product, filled to whole 16 bytes, stay
// under this many elements, so that a tile's extent is within a 31-bit buffer
// descriptor.
constexpr long kMaxPitch = 1L << 22;

// y = act(x W^T + bias) + residual; with `gated`, W = [Wg; Wu] of 2n rows and
// y = act(x Wg^T + bias[:n]) * (x Wu^T + bias[n:]).
// x and w: 16-byte aligned with pitches of whole 16 bytes and zeros behind k up
// to such.
struct Forward {
  int type, act;
  bool gated;
  long m, n, k;
  const void* x;
  long ldx;
  const void* w;
  long ldw;
  const void* bias;  // or null
  const void* res;   // or null
  long ldr;
  void* y;  // [m][n]
  // Pre-activations for the backward pass, or all null, with rows of `ldp`:
  //   linear   pre: 16 bits of the type, ldp a multiple of 8
  //   gated    pre and low: 24 bits, ldp a multiple of 16
  //   either   codes and scales: 8 bits, ldp a multiple of 32 (gated: 64) and
  //            ldp / 32 scales a row
  // The gated layer's up half begins ldp / 2 on.
  void* pre;
  unsigned char* low;
  unsigned char* codes;
  unsigned char* scales;
  long ldp;
  bool by_rows;  // few rows, on a kernel of their own
  TileChoice choice;
  float* part;  // [splits][m][n or 2n], with splits > 1
};
// Sets by_rows, or choice with splits >= 1.
void choose_forward(Forward& f);
void launch_linear_forward(const Forward& f, hipStream_t st);
void forward_tiles_bf16(const Forward& f, hipStream_t st);
void forward_tiles_fp16(const Forward& f, hipStream_t st);

// Activations in 8 bits: codes [m][ldc], scales [m][ldc / 32], ldc = n to a
// multiple of 32
struct Pack {
  int type;  // 2: fp32
  bool vec;  // 16-byte aligned rows, n in whole 16 bytes
  long m, n;
  void* x;
  long ldx;
  unsigned char* codes;
  unsigned char* scales;
  long ldc;
};
// The gradient of the pre-activations, and its sums over the rows for the
// bias: g = dy act'(pre), or [dy u act'(g), dy act(g)] for the gated layer.
struct Slope {
  int type, act;
  bool gated;
  bool vec_dy;  // n % 8 == 0, dy 16-byte aligned with a pitch of such
  long m, n;
  const void* dy;
  long ldy;
  const void* pre;  // as in Forward, or all null where act is none
  const unsigned char* low;
  const unsigned char* codes;
  const unsigned char* scales;
  long ldp;
  void* out;  // [m][ldo], zeros behind each half's n columns; or null
  long ldo;   // a multiple of 8; the gated layer's up half begins n on
  float* sums;   // [chunks][n or 2n], or null: the bias gradient's, to be
                 // added up
  int chunks;    // rows go to this many runs
  Pack input;    // with codes: to be unpacked by the same launch
  int strips;    // of 256 columns; launch_slope's
};
int slope_chunks(long m, long n);
void launch_slope(const Slope& s, hipStream_t st);

// out[m][n] = sum_k A(m,k) B(n,k) in the operands' type.  Operands 16-byte
// aligned with pitches of whole 16 bytes; an operand by k has k in whole 16
// bytes, its zeros included.
struct Matmul {
  long m, n, k;
  const void* a;
  long lda;
  const void* b;
  long ldb;
  void* out;    // [m][n]
  float* part;  // [splits][m][n], with splits > 1
  int splits;
};

// The linear layer's own, both operands by k, with splits > 1.
void split_tiles_bf16(const Matmul& p, Tile tile, hipStream_t st);
void split_tiles_fp16(const Matmul& p, Tile tile, hipStream_t st);

// dx = g W and dW = g^T x in one launch, either with m = 0 for none, and
// after them the sums of the bias gradient's runs (see Slope).
struct Backward {
  int type;
  Matmul dx;  // a = g by k, b = W by rows
  Matmul dw;  // a = g by rows, b = x by rows
  const float* sums;  // or null
  int chunks;
  long width;
  void* dbias;
  PairChoice choice;
};
void launch_backward(const Backward& b, hipStream_t st);
void backward_tiles_bf16(const Backward& b, hipStream_t st);
void backward_tiles_fp16(const Backward& b, hipStream_t st);

// Rows of `n` 16-bit values to rows of `ldo` >= n, zeros behind; none with
// m = 0.  Both in one launch.
struct Repack {
  const void* x;
  long ldx, m, n;
  void* out;
  long ldo;
};
void launch_repack(const Repack& a, const Repack& b, hipStream_t st);

void launch_pack(const Pack& p, hipStream_t st);
void launch_unpack(const Pack& p, hipStream_t st);  // zeros to ldx behind n

}  // namespace ff
