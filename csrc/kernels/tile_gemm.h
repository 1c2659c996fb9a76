// The tiled matrix product behind the linear and the gated layer, forward
// and backward: C[m][n] = sum_k A(m,k) B(n,k), bf16 or fp16 in, fp32 sums.
//
// Each operand lies either with k contiguous (element (r,k) at r*ld + k) or
// with its rows contiguous (element (r,k) at k*ld + r), so that one kernel
// serves all three products of a layer without a transposed copy:
//   y  = x W^T     A = x  by k      B = W by k
//   dx = g W       A = g  by k      B = W by rows
//   dW = g^T x     A = g  by rows   B = x by rows
//
// Four waves, 2 x 2, own a BM x BN tile; a wave owns (BM/2) x (BN/2) as
// 16x16x32 matrix instructions.  With 256 x 256 a wave reads (128 + 128) * 64
// values of LDS for 128 * 128 * 64 products: two thirds of what eight waves
// of 128 x 64 would read, and LDS reads, at 128 bytes a clock, are what runs
// next to the matrix pipe here.
//
// k goes in steps of 64, two of A and three of B in LDS: all of its 160 KB for
// one block of 256 x 256, or for two of 128 x 128.  A step has two halves, of
// 32 k's in registers each:
//   first half   products of the first 32 | reads of the second 32's fragments
//                                         | loads of B of step + 2
//   wait: own reads of this step done, own loads of the next landed; barrier
//   second half  products of the second 32 | reads of the next step's first
//                                          | loads of A of step + 2, over this
// so that every half has as many loads, which a CU takes 64 bytes a clock of,
// B has two halves or more to arrive in and A one or more.  Both in the second
// half (two of B in LDS) are 2% to 4% slower, steps of 32 in a ring of five
// 10% to 20%: 64-byte rows cost the L2 as much as 128-byte ones.
// 4096 x 4096 x 8192 takes 189 us with both operands by k (1458 TFLOP/s), 199
// with B and 204 with both by rows; without the loads it would be 168, and a
// loop of nothing but matrix instructions on random data runs at 2050 TFLOP/s
// for the card's power.
//
// Loads go from memory to LDS (16 bytes a lane) without passing registers,
// through buffer descriptors of the tile's own extent: what lies past the last
// row or the last k comes back as zero, and no index here passes 32 bits
// however large the operands are.
//
// LDS images are lane-linear (the loads write lane after lane), so bank
// conflicts are avoided by permuting which 16 bytes of a row a lane fetches.
//
// The matrix instruction's two operands are given as (B, A): a lane then
// holds four neighbouring columns n of one row m.  Two fragments side by side
// make it eight, for 16-byte stores: of B by k the rows are permuted within 32
// on their way into LDS; of B by rows, whose transposing reads need them in
// order to be free of bank conflicts, the results are exchanged between lanes
// (`eight`).
#pragma once

#include <type_traits>

#include "common.h"

namespace tile {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using i16x4 = __attribute__((ext_vector_type(4))) short;
using i16x8 = __attribute__((ext_vector_type(8))) short;

typedef __attribute__((address_space(3))) char lds_char;

// c += b a, in place.  Written as instructions because the compiler, given
// 256 accumulators a lane, moves them from register to register between
// steps; `AGPR` says which half of the register file holds them.  The
// compiler waits for the operands' loads; for the results the end
// of Product::run waits.
template <typename T, bool AGPR>
__device__ __forceinline__ void mfma(f32x4& c, i16x8 b, i16x8 a) {
  if constexpr (AGPR) {
    if constexpr (std::is_same<T, __bf16>::value)
      asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0"
                   : "+a"(c) : "v"(b), "v"(a));
    else
      asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0"
                   : "+a"(c) : "v"(b), "v"(a));
  } else {
    if constexpr (std::is_same<T, __bf16>::value)
      asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0"
                   : "+v"(c) : "v"(b), "v"(a));
    else
      asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0"
                   : "+v"(c) : "v"(b), "v"(a));
  }
}


// the same as a value, for the compiler to schedule
template <typename T>
__device__ __forceinline__ f32x4 mfma_value(i16x8 b, i16x8 a, f32x4 c) {
  using V = __attribute__((ext_vector_type(8))) T;
  if constexpr (std::is_same<T, __bf16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(V, b), __builtin_bit_cast(V, a), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(
        __builtin_bit_cast(V, b), __builtin_bit_cast(V, a), c, 0, 0, 0);
}

constexpr int BK = 64;
constexpr unsigned PAST = 0x80000000u;  // an offset past every descriptor

// Rows (or k's) begin at whole 16 bytes and end at such, with zeros behind the
// last k: an extent is taken to the next multiple of 8.
struct Operand {
  const void* p;
  long ld;    // elements from one row (or k) to the next
  long rows;  // extent along m or n
};

__device__ __forceinline__ long whole(long n) { return (n + 7) & ~7L; }

// One operand's tile: R rows by BK, 256 threads.
//   ROWS = false  LDS [R][64]: 128 bytes a row
//   ROWS = true   LDS [64][R]
// PERM: rows within each 32 are permuted (by k only, see above).
template <int R, bool ROWS, bool PERM>
struct Stage {
  static constexpr int BYTES = R * BK * 2;
  static constexpr int PASSES = BYTES / 4096;  // 16 bytes a thread
  static constexpr int RPP = 32;               // by k: rows a pass
  unsigned off[PASSES];
  unsigned chunk;  // by k: this lane's 16 bytes' first k

  // row0: the pass's first row, from the descriptor's base
  __device__ __forceinline__ void init(int tid, long ld, int pass, int row0) {
    if constexpr (ROWS) {
      int o = pass * 4096 + tid * 16;
      int k = o / (R * 2), b = o % (R * 2);
      off[pass] = (unsigned)(k * ld * 2) + (b ^ swizzle(k)) + row0 * 2;
    } else {
      const int q = tid >> 3;
      const int r = PERM ? ((q & 15) >> 2) * 8 + (q >> 4) * 4 + (q & 3) : q;
      chunk = ((tid & 7) ^ swap(q)) * 8;
      off[pass] = (unsigned)((row0 + r) * ld * 2) + chunk * 2;
    }
  }

  // By k: eight lanes read the same 16 bytes of eight rows, of which two fill
  // the 256 bytes that the banks hold side by side; from one such two to the
  // next the 16 bytes change places.
  static __device__ __forceinline__ int swap(int row) { return row & 7; }

  // By rows: half a wave's transposing read takes 32 bytes of the eight k's
  // 8 a + r, a < 2, r < 4; they go to eight different 32-byte spans of those
  // 256 bytes.  Where R is an odd multiple of 64, rows of odd k begin in the
  // middle of them already.
  static __device__ __forceinline__ int swizzle(int k) {
    return (R % 128 == 0 ? (k & 3) << 6 : (k & 2) << 5) | (k & 8) << 2;
  }
};

// A buffer descriptor: base, no stride, the extent in bytes (a load past it
// gives zeros), raw 32-bit data.
using Descriptor = __attribute__((ext_vector_type(4))) int;

__device__ __forceinline__ Descriptor descriptor(const void* p, long bytes) {
  const unsigned long a = (unsigned long)p;
  return Descriptor{(int)(unsigned)a, (int)((a >> 32) & 0xffff),
                    bytes < 0 ? 0 : (int)bytes, 0x00020000};
}

// Waits for all loads to LDS (LOADS > 0: but the last so many) and, if READS,
// for all reads of it; nothing is moved across.  As builtins, so that the
// compiler counts with them.
template <int LOADS, bool READS>
__device__ __forceinline__ void wait() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((LOADS & 15) | (LOADS >> 4) << 14 | 0x70 |
                             (READS ? 0 : 0xf00));
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// 16 bytes a lane from memory to LDS at `dst` + 16 lane; `dst` is the wave's.
// As an instruction, because before a transposing read of LDS the compiler
// waits for every such load that it knows of.  It has no register to write,
// and `wait` is what waits for it.  M0, which it takes the place from, is the
// compiler's only around instructions that these kernels do not have.
__device__ __forceinline__ void load_lds(Descriptor r, lds_char* dst,
                                         unsigned off, int soff) {
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, %3 offen lds"
      :
      : "s"((unsigned)(unsigned long)dst), "v"(off), "s"(r), "s"(soff));
}

// Blocks go round the 8 XCDs by their number; giving each XCD a run of
// consecutive tiles, and ordering the tiles in strips of 8 tile rows, keeps
// the operands that neighbours share in that XCD's L2.
__device__ __forceinline__ void tile_of(int id, int total, int mt, int nt,
                                        int& tm, int& tn) {
  const int q = total >> 3, r = total & 7, xcd = id & 7, pos = id >> 3;
  id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + pos;
  const int strip = 8 * nt, first = id / strip * 8;
  const int high = mt - first < 8 ? mt - first : 8;
  tm = first + id % strip % high;
  tn = id % strip / high;
}

// The product of one tile: acc[i][j] is a 16 x 16 block of rows wm + 16 i and,
// with its neighbour, columns wn + 32 (j / 2) + 0..31; lane l holds row l % 16
// of it.  `eight` gives its eight neighbouring columns of the two, which begin
// at `column`.
//
// SPLITB: B's tile is two runs of BN/2 rows, `second` rows apart, one after
// the other in each wave's half of the tile (the gated layer's two weights).
template <typename T, int BM, int BN, bool AROWS, bool BROWS, bool SPLITB>
struct Product {

  static constexpr int WM = BM / 2, WN = BN / 2;
  static constexpr int FM = WM / 16, FN = WN / 16;
  static constexpr bool AGPR = FM * FN >= 32;
  using SA = Stage<BM, AROWS, false>;
  using SB = Stage<BN, BROWS, true>;
  static constexpr int LDS = 2 * SA::BYTES + 3 * SB::BYTES;
  static_assert(!SPLITB || (!BROWS && WN / 2 >= SB::RPP), "whole passes");

  f32x4 acc[FM][FN];

  static __device__ __forceinline__ int column(int lane) {
    const int g = lane >> 4;
    return BROWS ? (g & 1) * 16 + (g >> 1) * 8 : g * 8;
  }

  __device__ __forceinline__ void eight(int i, int pair, float* v) const {
    const f32x4 a = acc[i][2 * pair], b = acc[i][2 * pair + 1];
#pragma unroll
    for (int r = 0; r < 4; r++) {
      if constexpr (BROWS) {
        // lanes 16..31 of a change places with lanes 0..15 of b, and 48..63
        // with 32..47
        const auto s = __builtin_amdgcn_permlane16_swap(
            __float_as_uint(a[r]), __float_as_uint(b[r]), false, false);
        v[r] = __uint_as_float(s[0]);
        v[4 + r] = __uint_as_float(s[1]);
      } else {
        v[r] = a[r];
        v[4 + r] = b[r];
      }
    }
  }

  // The loads of one operand, a step at a time.  By k the descriptor stays and
  // k is the loads' scalar offset: rows are told apart by the lanes' offsets
  // alone, k's by `in`.  By rows the descriptor moves on, over what is left.
  template <bool ROWS>
  struct Feed {
    const char* p;
    long rest;  // bytes from p
    long step;  // bytes a step
    int k;      // bytes

    __device__ __forceinline__ void init(const Operand& o, long r0, int rows,
                                         long k0, long k1) {
      const long left = o.rows - r0;
      if constexpr (ROWS) {
        p = (const char*)o.p + (k0 * o.ld + r0) * 2;
        rest = ((k1 - k0 - 1) * o.ld + whole(left)) * 2;
        step = BK * o.ld * 2;
      } else {
        p = (const char*)o.p + (r0 * o.ld + k0) * 2;
        rest = (((left < rows ? left : rows) - 1) * o.ld + whole(k1 - k0)) * 2;
        step = BK * 2;
      }
      k = 0;
    }
    __device__ __forceinline__ Descriptor get() const {
      // an extent past 2^31 - 1 is as good as that: a step's offsets are less
      const long most = 0x7fffffffL;
      return descriptor(p, rest > most ? most : rest);
    }
    __device__ __forceinline__ void next() {
      if constexpr (ROWS) {
        p += step;
        rest -= step;
      } else {
        k += BK * 2;
      }
    }
  };

  __device__ __forceinline__ void run(char* smem_, const Operand& A,
                                      const Operand& B, long m0, long n0,
                                      long k0, long k1, long second) {
    lds_char* smem = (lds_char*)smem_;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = (wid >> 1) * WM, wn = (wid & 1) * WN;

    SA sa;
    SB sb;
#pragma unroll
    for (int p = 0; p < SA::PASSES; p++) sa.init(tid, A.ld, p, AROWS ? 0 : p * SA::RPP);
#pragma unroll
    for (int p = 0; p < SB::PASSES; p++) {
      int r = p * SB::RPP;
      if constexpr (SPLITB) r = (r / WN) * (WN / 2) + r % (WN / 2);
      sb.init(tid, B.ld, p, BROWS ? 0 : r);
    }

    Feed<AROWS> fa;
    Feed<BROWS> fb, fb2;
    constexpr int RB = SPLITB ? BN / 2 : BN;
    fa.init(A, m0, BM, k0, k1);
    fb.init(B, n0, RB, k0, k1);
    if constexpr (SPLITB) {
      fb2 = fb;
      fb2.p += second * B.ld * 2;
    }
    const int steps = (int)((k1 - k0 + BK - 1) / BK);
    const int extent = (int)(k1 - k0);
    int ka = 0, kb = 0;  // the next loads' first k
    lds_char* const ldsa = smem;
    lds_char* const ldsb = smem + 2 * SA::BYTES;

    // One operand's loads of its next step, some at a time.  Past the last
    // step all lanes' offsets lie outside: zeros, which nothing reads.
    struct Source {
      Descriptor r, r2;
      bool in;
    };
    auto source_a = [&]() {
      Source s;
      s.r = fa.get();
      s.in = AROWS || (int)sa.chunk < extent - ka;
      return s;
    };
    auto source_b = [&]() {
      Source s;
      s.r = fb.get();
      if constexpr (SPLITB) s.r2 = fb2.get();
      s.in = BROWS || (int)sb.chunk < extent - kb;
      return s;
    };
    auto load_a = [&](const Source& s, lds_char* to, int p) {
      load_lds(s.r, to + wid * 1024 + p * 4096, s.in ? sa.off[p] : PAST, fa.k);
      if (p == SA::PASSES - 1) {
        fa.next();
        ka += BK;
      }
    };
    auto load_b = [&](const Source& s, lds_char* to, int p) {
      const bool up = SPLITB && (p * SB::RPP) % WN >= WN / 2;
      load_lds(up ? s.r2 : s.r, to + wid * 1024 + p * 4096,
               s.in ? sb.off[p] : PAST, fb.k);
      if (p == SB::PASSES - 1) {
        fb.next();
        kb += BK;
      }
    };

    // ---- fragment addresses --------------------------------------------
    const int g = lane >> 4, l = lane & 15;
    const int trk = g * 8 + (l >> 2);  // by rows: this lane's k
    // by k one address serves all fragments, 16 rows or 2048 bytes apart
    unsigned aoff[AROWS ? FM : 1], boff[BROWS ? FN : 1];
    if constexpr (AROWS) {
#pragma unroll
      for (int i = 0; i < FM; i++)
        aoff[i] = trk * (BM * 2) +
                  (((wm + i * 16) * 2 + (l & 3) * 8) ^ SA::swizzle(trk));
    } else {
      aoff[0] = (wm + l) * 128 + ((g ^ SA::swap(l)) << 4);
    }
    if constexpr (BROWS) {
#pragma unroll
      for (int j = 0; j < FN; j++)
        boff[j] = trk * (BN * 2) +
                  (((wn + j * 16) * 2 + (l & 3) * 8) ^ SB::swizzle(trk));
    } else {
      boff[0] = (wn + l) * 128 + ((g ^ SB::swap(l)) << 4);
    }

    auto tr = [&](lds_char* p, int half) {  // four more k's: `half` bytes on
      typedef __attribute__((address_space(3))) i16x4 lds_v4;
      i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4*)p);
      i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4*)(p + half));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    typedef __attribute__((address_space(3))) i16x8 lds_v8;

    auto read_a = [&](i16x8(&f)[FM], int i, lds_char* t, int kk) {
      if constexpr (AROWS)
        f[i] = tr(t + aoff[i] + kk * 64 * BM, 8 * BM);
      else
        f[i] = *(lds_v8*)(t + (aoff[0] ^ (kk << 6)) + i * 2048);
    };
    auto read_b = [&](i16x8(&f)[FN], int j, lds_char* t, int kk) {
      if constexpr (BROWS)
        f[j] = tr(t + boff[j] + kk * 64 * BN, 8 * BN);
      else
        f[j] = *(lds_v8*)(t + (boff[0] ^ (kk << 6)) + j * 2048);
    };
    // The products of 32 k's, of ua and ub.  A matrix instruction keeps its
    // pipe busy for 16 clocks and the wave for 4: what else there is to issue
    // goes in between, one at a time.  That is the next 32's reads into na and
    // nb (B's fragments first, which every row of blocks needs; none in the
    // last quarter, so that the wait finds them done) and one operand's loads.
    constexpr int READS = FM + FN, SLOTS = FM * FN;
    auto half = [&](const i16x8(&ua)[FM], const i16x8(&ub)[FN],
                    i16x8(&na)[FM], i16x8(&nb)[FN], lds_char* ra,
                    lds_char* rb, int kk, bool b_loads, lds_char* to) {
      const int loads = b_loads ? SB::PASSES : SA::PASSES;
      const Source src = b_loads ? source_b() : source_a();
#pragma unroll
      for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) {
          const int slot = i * FN + j;
          mfma<T, AGPR>(acc[i][j], ub[j], ua[i]);
          __builtin_amdgcn_sched_barrier(0);
          // the reads and loads that fall due by the end of this slot
#pragma unroll
          for (int x = slot * READS * 4 / (SLOTS * 3);
               x < (slot + 1) * READS * 4 / (SLOTS * 3) && x < READS;
               x++) {
            if (x < FN)
              read_b(nb, x, rb, kk);
            else
              read_a(na, x - FN, ra, kk);
          }
#pragma unroll
          for (int q = slot * loads / SLOTS; q < (slot + 1) * loads / SLOTS;
               q++) {
            if (b_loads)
              load_b(src, to, q);
            else
              load_a(src, to, q);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
    };

#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
      for (int j = 0; j < FN; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    i16x8 a0[FM], b0[FN], a1[FM], b1[FN];
#pragma unroll
    for (int n = 0; n < 2; n++) {
      const Source rb = source_b();
#pragma unroll
      for (int p = 0; p < SB::PASSES; p++)
        load_b(rb, ldsb + n * SB::BYTES, p);
      const Source ra = source_a();
#pragma unroll
      for (int p = 0; p < SA::PASSES; p++)
        load_a(ra, ldsa + n * SA::BYTES, p);
    }
    wait<SA::PASSES + SB::PASSES, false>();  // step 0 has landed
    barrier();
#pragma unroll
    for (int j = 0; j < FN; j++) read_b(b0, j, ldsb, 0);
#pragma unroll
    for (int i = 0; i < FM; i++) read_a(a0, i, ldsa, 0);
    wait<63, true>();
    asm volatile("s_nop 7");  // the accumulators' zeros
    lds_char* pa = ldsa;      // step s's buffers
    lds_char* pb = ldsb;
    lds_char* const last = ldsb + 2 * SB::BYTES;
    for (int s = 0; s < steps; s++) {
      lds_char* const qa = pa == ldsa ? ldsa + SA::BYTES : ldsa;
      lds_char* const qb = pb == last ? ldsb : pb + SB::BYTES;
      half(a0, b0, a1, b1, pa, pb, 1, true, qb == last ? ldsb : qb + SB::BYTES);
      wait<SB::PASSES, true>();
      barrier();
      half(a1, b1, a0, b0, qa, qb, 0, false, pa);
      wait<63, true>();  // the reads ended rows ago; here they are counted
      pa = qa;
      pb = qb;
    }
    // No load may write LDS after this: the block's LDS is another's once it
    // ends.  And the last products' results: 4 passes of 4 clocks each at
    // least have to go by before another instruction reads them.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_nop 15\n\ts_nop 15" :::
                 "memory");
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
      for (int j = 0; j < FN; j++) {
        if constexpr (AGPR)
          asm volatile("" : "+a"(acc[i][j]));
        else
          asm volatile("" : "+v"(acc[i][j]));
      }
  }
};

}  // namespace tile
