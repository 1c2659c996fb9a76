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
// 4096 x 4096 x 8192 takes 174 us with both operands by k (1582 TFLOP/s), 186
// with B and 189 with both by rows; on another card, in a row of 40, 188 (1461
// TFLOP/s), 190 and 195, where the library takes 210.  Without the loads the
// 174 were 168, and a loop of nothing but matrix instructions on random data
// runs at 2050 TFLOP/s: the card's power is the bound, the clock falls as the
// pipe fills.
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
//
// A wave fills a run of LDS, 1024 bytes a pass, so that four passes have one
// LDS base and differ in the instruction's own offset.  That offset moves the
// address in memory as well: `off` is so much less, and the descriptor's base
// LEAD bytes before the operand, which no lane's offset reaches.
constexpr int LEAD = 3 * 1024;

template <int R, bool ROWS, bool PERM>
struct Stage {
  static constexpr int BYTES = R * BK * 2;
  static constexpr int PASSES = BYTES / 4096;  // 16 bytes a thread
  unsigned off[PASSES];
  unsigned chunk;  // by k: this lane's 16 bytes' first k

  // HALVES: two runs of R / 2 rows, which the waves take in turns; offsets
  // count from the first row of the wave's run
  template <bool HALVES>
  __device__ __forceinline__ void init(int wid, int lane, long ld) {
#pragma unroll
    for (int p = 0; p < PASSES; p++) {
      const int o = (wid * PASSES + p) * 1024 + lane * 16;
      unsigned at;
      if constexpr (ROWS) {
        const int k = o / (R * 2), b = o % (R * 2);
        at = (unsigned)(k * ld * 2) + (b ^ swizzle(k));
      } else {
        const int row = o >> 7, q = row & 31;
        int r = (row & ~31) +
                (PERM ? ((q & 15) >> 2) * 8 + (q >> 4) * 4 + (q & 3) : q);
        if constexpr (HALVES) r = (wid >> 1) * (R / 4) + r % (R / 4);
        chunk = ((lane & 7) ^ swap(row)) * 8;
        at = (unsigned)(r * ld * 2) + chunk * 2;
      }
      off[p] = at + LEAD - (p & 3) * 1024;
    }
  }

  // The last k's: lanes past them load nothing.  Once is enough for a step;
  // from then on they stay past.
  __device__ __forceinline__ void cut(int left) {
#pragma unroll
    for (int p = 0; p < PASSES; p++)
      off[p] = (int)chunk < left ? off[p] : PAST;
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

__device__ __forceinline__ Descriptor descriptor(const char* p, int bytes) {
  const unsigned long a = (unsigned long)(p - LEAD);
  return Descriptor{(int)(unsigned)a, (int)((a >> 32) & 0xffff), bytes,
                    0x00020000};
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

// 16 bytes a lane from memory to LDS at M0 + 1024 PASS + 16 lane.  As an
// instruction, because before a transposing read of LDS the compiler waits for
// every such load that it knows of.  It has no register to write, and `wait`
// is what waits for it.  M0 is the compiler's only around instructions that
// these kernels do not have; one other instruction has to lie between `set_m0`
// and the load.  As every instruction between two matrix instructions counts
// (one idle one more to each load costs 2% to 8%), M0 is set for four loads
// and their lanes' offsets are ready.
__device__ __forceinline__ void set_m0(lds_char* dst) {
  asm volatile("s_mov_b32 m0, %0" : : "s"((unsigned)(unsigned long)dst)
               : "m0");
}

template <int AT>
__device__ __forceinline__ void load_lds_at(Descriptor r, unsigned off,
                                            int soff) {
  asm volatile("buffer_load_dwordx4 %0, %1, %2 offen offset:%3 lds"
               : : "v"(off), "s"(r), "s"(soff), "n"(AT));
}

__device__ __forceinline__ void load_lds(Descriptor r, unsigned off, int soff,
                                         int pass) {
  switch (pass & 3) {
    case 0: return load_lds_at<0>(r, off, soff);
    case 1: return load_lds_at<1024>(r, off, soff);
    case 2: return load_lds_at<2 * 1024>(r, off, soff);
    default: return load_lds_at<3 * 1024>(r, off, soff);
  }
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
  static_assert(!SPLITB || !BROWS, "the weights lie by k");

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
  // alone, k's by `cut`.  By rows the descriptor moves on, over a step's k's.
  template <typename S, bool ROWS>
  struct Feed {
    const char* p;
    long step;             // bytes a step
    int full, part, soff;  // a step's extent, the last step's
    int left;              // k's from this step on
    Descriptor d;

    __device__ __forceinline__ void init(const Operand& o, long r0, int rows,
                                         long k0, long k1) {
      const long ext = whole(o.rows - r0);
      left = (int)(k1 - k0);
      soff = 0;
      if constexpr (ROWS) {
        p = (const char*)o.p + (k0 * o.ld + r0) * 2;
        step = BK * o.ld * 2;
        full = (int)(((BK - 1) * o.ld + ext) * 2) + LEAD;
        part = (int)((((left - 1) % BK) * o.ld + ext) * 2) + LEAD;
      } else {
        const long has = o.rows - r0;
        p = (const char*)o.p + (r0 * o.ld + k0) * 2;
        const long bytes =
            (((has < rows ? has : rows) - 1) * o.ld + whole(left)) * 2 + LEAD;
        // rows past the last: no extent
        d = descriptor(p, has > 0 ? (int)bytes : 0);
      }
    }
    // to be called before a step's loads
    __device__ __forceinline__ void begin(S& s) {
      if constexpr (ROWS) {
        d = descriptor(p, left >= BK ? full : left > 0 ? part : 0);
      } else {
        if (left < BK) s.cut(left);
      }
    }
    __device__ __forceinline__ void next() {
      left -= BK;
      if constexpr (ROWS) p += step;
      else soff += BK * 2;
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
    sa.template init<false>(wid, lane, A.ld);
    sb.template init<SPLITB>(wid, lane, B.ld);
    Feed<SA, AROWS> fa;
    Feed<SB, BROWS> fb;
    fa.init(A, m0, BM, k0, k1);
    {
      // of two runs, odd waves take the second
      Operand o = B;
      if (SPLITB && (wid & 1)) o.p = (const char*)B.p + second * B.ld * 2;
      fb.init(o, n0, SPLITB ? BN / 2 : BN, k0, k1);
    }
    const int steps = (int)((k1 - k0 + BK - 1) / BK);
    lds_char* const ldsa = smem;
    lds_char* const ldsb = smem + 2 * SA::BYTES;

    // Load p of an operand's step, into the buffer `to`; M0 is set for four
    // of them, one matrix instruction (or an idle one) before.
    auto base_a = [&](lds_char* to, int p) {
      set_m0(to + wid * (SA::PASSES * 1024) + (p & ~3) * 1024);
    };
    auto base_b = [&](lds_char* to, int p) {
      set_m0(to + wid * (SB::PASSES * 1024) + (p & ~3) * 1024);
    };
    auto load_a = [&](int p) {
      load_lds(fa.d, sa.off[p], fa.soff, p);
      if (p == SA::PASSES - 1) fa.next();
    };
    auto load_b = [&](int p) {
      load_lds(fb.d, sb.off[p], fb.soff, p);
      if (p == SB::PASSES - 1) fb.next();
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
      if (b_loads) {
        fb.begin(sb);
        base_b(to, 0);
      } else {
        fa.begin(sa);
        base_a(to, 0);
      }
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
            if (b_loads) {
              load_b(q);
              if ((q & 3) == 3 && q + 1 < loads) base_b(to, q + 1);
            } else {
              load_a(q);
              if ((q & 3) == 3 && q + 1 < loads) base_a(to, q + 1);
            }
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
      fb.begin(sb);
#pragma unroll
      for (int p = 0; p < SB::PASSES; p++) {
        if ((p & 3) == 0) {
          base_b(ldsb + n * SB::BYTES, p);
          asm volatile("s_nop 0");
        }
        load_b(p);
      }
      fa.begin(sa);
#pragma unroll
      for (int p = 0; p < SA::PASSES; p++) {
        if ((p & 3) == 0) {
          base_a(ldsa + n * SA::BYTES, p);
          asm volatile("s_nop 0");
        }
        load_a(p);
      }
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
