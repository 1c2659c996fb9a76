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
// k goes in steps of 64 through two LDS buffers.  A step is two halves of 32:
//   first half   read the second half's fragments   | products of the first
//   wait: own loads of the next step landed, own reads of this buffer done
//   barrier
//   second half  load step + 2 into this buffer, read the next step's first
//                fragments from the other one       | products of the second
// so a load has a whole step's products to arrive in, and one barrier a step
// is enough.  Loads go from memory to LDS (16 bytes a lane) without passing
// registers, through buffer descriptors of the tile's own extent: what lies
// past the last row or the last k comes back as zero, and no index here
// passes 32 bits however large the operands are.
//
// LDS images are lane-linear (the loads write lane after lane), so bank
// conflicts are avoided by permuting which 16 bytes of a row a lane fetches.
//
// The matrix instruction's two operands are given as (B, A): a lane then
// holds four neighbouring columns n of one row m.  B's rows are permuted
// within 32 (on the way into LDS, or in the read for the by-rows layout) so
// that two fragments side by side make it eight: 16-byte stores.
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
// PERM: rows within each 32 are permuted (see above; by-k layout only, the
// by-rows layout permutes in its reads).
template <int R, bool ROWS, bool PERM>
struct Stage {
  static constexpr int PASSES = R / 32;   // 4096 bytes a pass
  static constexpr int BYTES = R * BK * 2;
  static constexpr int KPP = 2048 / R;    // by rows: k's a pass
  unsigned off[PASSES];
  unsigned chunk;  // by k: this lane's 16 bytes' first k

  // row0 counts from the descriptor's base
  __device__ __forceinline__ void init(int tid, long ld, int pass, int row0) {
    if constexpr (ROWS) {
      int o = pass * 4096 + tid * 16;
      int k = o / (R * 2), b = o % (R * 2);
      off[pass] = (unsigned)(k * ld * 2) + (b ^ swizzle(k)) + row0 * 2;
    } else {
      int q = tid >> 3, s = tid & 7;
      int r = PERM ? ((q & 15) >> 2) * 8 + (q >> 4) * 4 + (q & 3) : q;
      chunk = (s ^ (q & 7)) * 8;
      off[pass] = (unsigned)((row0 + r) * ld * 2) + chunk * 2;
    }
  }

  static __device__ __forceinline__ int swizzle(int k) {
    // four k's at the same 32 bytes of a row go to four 64-byte spans
    return R >= 128 ? (k & 3) << 6 : (k & 2) << 5;
  }
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t descriptor(const void* p,
                                                             long bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0,
                                           bytes < 0 ? 0 : (int)bytes,
                                           0x00020000);
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

__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t r,
                                         lds_char* dst, unsigned off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      r, (__attribute__((address_space(3))) void*)dst, 16, off, 0, 0, 0);
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

// The product of one tile: acc[i][j] is the 16 x 16 block of rows
// wm + 16 i and columns (a pair of j's: 32) wn + 32 (j / 2); lane l holds row
// l % 16, columns 8 (l / 16) + 4 (j % 2) + 0..3 of it.
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
  static constexpr int BUF = SA::BYTES + SB::BYTES;
  static constexpr int LDS = 2 * BUF;

  f32x4 acc[FM][FN];

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
    for (int p = 0; p < SA::PASSES; p++)
      sa.init(tid, A.ld, p, AROWS ? 0 : p * 32);
#pragma unroll
    for (int p = 0; p < SB::PASSES; p++) {
      int r = p * 32;
      if constexpr (SPLITB) r = (r / WN) * (WN / 2) + r % (WN / 2);
      sb.init(tid, B.ld, p, BROWS ? 0 : r);
    }

    const char* ap = (const char*)A.p + (AROWS ? m0 : m0 * A.ld) * 2;
    const char* bp = (const char*)B.p + (BROWS ? n0 : n0 * B.ld) * 2;
    const long am = A.rows - m0, bn = B.rows - n0;

    const int steps = (int)((k1 - k0 + BK - 1) / BK);

    // What step s loads; past the last step descriptors of no extent, whose
    // loads bring zeros that nothing reads.
    struct Source {
      __amdgpu_buffer_rsrc_t a, b, b2;
      bool in_a, in_b;  // by k: whether this lane's 16 bytes lie before k1
    };
    auto source = [&](int s) {
      const long k = k0 + (long)s * BK;
      const long left = k1 - k;
      const bool any = left > 0;
      constexpr int RB = SPLITB ? BN / 2 : BN;
      const long mk = left < BK ? left : BK;
      const long ab = AROWS ? (mk - 1) * A.ld + whole(am)
                            : ((am < BM ? am : BM) - 1) * A.ld + whole(left);
      const long bb = BROWS ? (mk - 1) * B.ld + whole(bn)
                            : ((bn < RB ? bn : RB) - 1) * B.ld + whole(left);
      Source r;
      r.a = descriptor(ap + (AROWS ? k * A.ld : k) * 2, any ? ab * 2 : 0);
      r.b = descriptor(bp + (BROWS ? k * B.ld : k) * 2, any ? bb * 2 : 0);
      if constexpr (SPLITB)
        r.b2 = descriptor(bp + (second * B.ld + k) * 2, any ? bb * 2 : 0);
      r.in_a = AROWS || (long)sa.chunk < left;
      r.in_b = BROWS || (long)sb.chunk < left;
      return r;
    };
    constexpr int LOADS = SA::PASSES + SB::PASSES;
    auto load = [&](const Source& r, int buf, int p) {
      lds_char* to = smem + buf * BUF + wid * 1024;
      if (p < SA::PASSES) {
        load_lds(r.a, to + p * 4096, r.in_a ? sa.off[p] : PAST);
      } else {
        const int q = p - SA::PASSES;
        const bool up = SPLITB && (q * 32) % WN >= WN / 2;
        load_lds(up ? r.b2 : r.b, to + SA::BYTES + q * 4096,
                 r.in_b ? sb.off[q] : PAST);
      }
    };

    // ---- fragment addresses --------------------------------------------
    const int g = lane >> 4, l = lane & 15;
    unsigned abase, bbase;
    if constexpr (AROWS) {
      const int k = g * 8 + (l >> 2);
      abase = k * (BM * 2) + ((wm * 2 + (l & 3) * 8) ^ SA::swizzle(k));
    } else {
      abase = (wm + l) * 128 + ((g ^ (l & 7)) << 4);
    }
    if constexpr (BROWS) {
      const int k = g * 8 + (l >> 2);
      bbase = k * (BN * 2) + ((wn * 2 + (l & 3) * 16) ^ SB::swizzle(k));
    } else {
      bbase = (wn + l) * 128 + ((g ^ (l & 7)) << 4);
    }

    auto tr = [&](lds_char* p, int half) {  // four more k's: `half` bytes on
      typedef __attribute__((address_space(3))) i16x4 lds_v4;
      i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4*)p);
      i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4*)(p + half));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    typedef __attribute__((address_space(3))) i16x8 lds_v8;

    auto read_a = [&](i16x8(&f)[FM], int i, int buf, int kk) {
      lds_char* t = smem + buf * BUF;
      if constexpr (AROWS)
        // 32 bytes a fragment: bit 5 adds, bits 6 and 7 are the swizzle's
        f[i] = tr(t + (abase ^ ((i >> 1) << 6)) + (i & 1) * 32 +
                      kk * 32 * BM * 2,
                  4 * BM * 2);
      else
        f[i] = *(lds_v8*)(t + (abase ^ (kk << 6)) + i * 2048);
    };
    auto read_b = [&](i16x8(&f)[FN], int j, int buf, int kk) {
      lds_char* t = smem + buf * BUF + SA::BYTES;
      if constexpr (BROWS)
        f[j] = tr(t + (bbase ^ ((j >> 1) << 6)) + (j & 1) * 8 +
                      kk * 32 * BN * 2,
                  4 * BN * 2);
      else
        f[j] = *(lds_v8*)(t + (bbase ^ (kk << 6)) + j * 2048);
    };
    // Half a step: the products of fa and fb, row of blocks by row, with the
    // next half's reads into na and nb and, after the barrier, the loads of
    // step + 2 between the rows: B's fragments first, which every row needs.
    constexpr int READS = FM + FN;
    auto half = [&](const i16x8(&fa)[FM], const i16x8(&fb)[FN],
                    i16x8(&na)[FM], i16x8(&nb)[FN], int rbuf, int rkk,
                    bool loads, const Source& r, int lbuf) {
      constexpr int RPG = (READS + FM - 3) / (FM > 2 ? FM - 2 : 1);
      constexpr int LPG = (LOADS + FM - 1) / FM;
#pragma unroll
      for (int i = 0; i < FM; i++) {
#pragma unroll
        for (int q = 0; q < RPG; q++) {
          const int x = i * RPG + q;
          if (x < FN)
            read_b(nb, x, rbuf, rkk);
          else if (x < READS)
            read_a(na, x - FN, rbuf, rkk);
        }
        if (loads) {
#pragma unroll
          for (int q = 0; q < LPG; q++)
            if (i * LPG + q < LOADS) load(r, lbuf, i * LPG + q);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < FN; j++)
          mfma<T, AGPR>(acc[i][j], fb[j], fa[i]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };

#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
      for (int j = 0; j < FN; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    i16x8 a0[FM], b0[FN], a1[FM], b1[FN];
    {
      const Source r0 = source(0), r1 = source(1);
#pragma unroll
      for (int p = 0; p < LOADS; p++) load(r0, 0, p);
#pragma unroll
      for (int p = 0; p < LOADS; p++) load(r1, 1, p);
    }
    // step 0 has landed once only step 1's loads are under way
    wait<LOADS, false>();
    barrier();
#pragma unroll
    for (int j = 0; j < FN; j++) read_b(b0, j, 0, 0);
#pragma unroll
    for (int i = 0; i < FM; i++) read_a(a0, i, 0, 0);
    wait<63, true>();
    asm volatile("s_nop 7");  // the accumulators' zeros
    for (int s = 0; s < steps; s++) {
      const int buf = s & 1;
      const Source next = source(s + 2);
      half(a0, b0, a1, b1, buf, 1, false, next, buf);
      wait<0, true>();
      barrier();
      half(a1, b1, a0, b0, buf ^ 1, 0, true, next, buf);
      wait<63, true>();  // the reads ended rows ago; here they are counted
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
