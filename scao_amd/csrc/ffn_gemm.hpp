// Tiled matrix products of the gated feed-forward block on gfx950's bf16 and
// fp16 matrix cores, with the block's epilogues.
//
//   C[m][n] = sum over segments s and k of A_s[m][k] B_s[n][k]
//
// An operand is stored either with k contiguous ("rows": element (r, k) at
// r*ld + k) or with r contiguous ("cols": k*ld + r); the six products of the
// block's forward and backward pass need rows x rows, rows x cols and cols x
// cols.  Segments add products of different operands of one shape: da Wg + db
// Wu, and the six partial products of an fp32 product on bf16 cores.
//
// A workgroup owns a BM x BN tile of C and walks k in steps of 64.  Each step's
// two tiles go from global memory to LDS without passing registers (16 bytes a
// lane), A's into the third of three stages while two are in use, B's into the
// other of two (a third one does not fit, and gains nothing for 256 x 256 tiles;
// A's does 3% for 128 x 128).  The buffer descriptor's bound and an out-of-range
// lane offset give zeros outside the operands, so no edge needs a branch.
//
// What bounds it: on random data the chip's power, with zeros 1810 TFLOP/s where
// random bf16 reach 1410 (8192^3, 256 x 256 tiles; rows x rows 1410-1430, rows x
// cols 1390, cols x cols 1400; 128 x 128 tiles 1140).  Before that it was the
// order of issue.  A wave's loads and LDS reads queued ahead of its products left
// the matrix cores idle (1276; with no loads at all 1716), so every row of
// products carries its share of both (half()), and all loads in the first half
// of the rows cost 6% again.  Four waves of 128 x 128 products instead of eight of
// 128 x 64 halve the LDS reads, but leave one wave a SIMD (1237); 32 x 32 x 16
// products are faster on half of the chip (930 against 890 TFLOP/s on 128 CUs)
// and slower on all of it (1285).
//
// LDS layout.  The direct load writes lane l's 16 bytes at l*16, so tiles are
// permuted by choosing which 16 bytes a lane fetches:
//   rows: a row's 64 k are 8 chunks of 16 bytes; chunk c of row r lies at c ^
//         (r & 7), so that the 16 rows a fragment read touches spread over all
//         banks;
//   cols: a k's R elements are R/16 chunks of 32 bytes; chunk c of k lies at
//         c ^ f(k), f(k) = (k & 3) | (k >> 3 & 1) << 2: a transposing read takes
//         32 bytes of 16 different k.
#pragma once

#include "../../include/scao_train.h"
#include "scao_common.hpp"

namespace scao {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lchar;
typedef __attribute__((address_space(3))) v4s lv4s;
typedef __attribute__((address_space(3))) v8s lv8s;

constexpr int FFN_BK = 64;
constexpr int FFN_MAX_SEG = 12;

enum { ROWS = 0, COLS = 1 };

// one 16x16x32 product: lane l supplies P[l%16][8*(l/16)+e] and Q[l%16][8*(l/16)+e];
// element r of the result is the product of P's row 4*(l/16)+r and Q's row l%16
template <bool F16>
__device__ __forceinline__ v4f mma(v8s p, v8s q, v4f c) {
  if (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, p),
                                                  __builtin_bit_cast(v8h, q), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, p),
                                                 __builtin_bit_cast(v8bf, q), c, 0, 0, 0);
}

// 16 bytes a lane from global memory to LDS at lds + 16*lane.  The compiler
// neither counts this load nor waits for it: wait_loads does, which it cannot
// pass.  Nor does it look into the block for the waits that the instructions
// need of each other: one after m0 is written before a load uses it, five after a
// vector instruction (readfirstlane) has written an operand's scalar register.
// (m0 cannot be listed as changed; the compiler itself has no use for it here:
// gfx950's LDS instructions do not read it.)
__device__ __forceinline__ void load_lds(v4i rsrc, uint32_t lds, uint32_t voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(
                   __builtin_amdgcn_readfirstlane(lds)),
               "v"(voff), "s"(rsrc));
}
// all but the last N loads of this wave have arrived in LDS and every LDS read
// of it has been answered, and every other wave says the same
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

constexpr uint32_t OUT_OF_RANGE = 0x80000000u;

__device__ __forceinline__ v4i buffer_of(const void* p, int64_t bytes) {
  const uint64_t a = (uint64_t)(uintptr_t)p;
  const int64_t n = bytes < 0 ? 0 : bytes > 0x7fffffff ? 0x7fffffff : bytes;
  v4i r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  r[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32) & 0xffff);
  r[2] = __builtin_amdgcn_readfirstlane((int)n);
  r[3] = 0x00020000;
  return r;
}

// One operand's share of a step: R rows (of C's dimension) by 64 k, 16-bit.  WORDS 2:
// by 32 k of two words each, the lower ones behind the higher ones of all 32 k; in
// memory they lie `low` elements behind them.
template <int L, int R, int NW, int WORDS = 1>
struct Tile {
  static constexpr int BYTES = R * FFN_BK * 2;
  static constexpr int LOADS = BYTES / 1024 / NW;   // per wave and step
  static constexpr int KROW = R * 2;                // cols: bytes of one k
  static_assert(BYTES % (1024 * NW) == 0, "whole loads a wave");

  // byte offset, relative to the step's origin, of what lane `lane` of load i
  // of wave w fetches
  static __device__ __forceinline__ uint32_t offset(int i, int w, int lane, int64_t ld,
                                                    int low = 0) {
    const int at = (i * NW + w) * 1024 + lane * 16;
    if (L == ROWS) {
      const int r = at / 128, c = (at % 128) / 16 ^ (r & 7);
      if (WORDS == 2) return (uint32_t)(r * ld * 2 + (c & 3) * 16 + (c >> 2) * low * 2);
      return (uint32_t)(r * ld * 2 + c * 16);
    }
    const int k = at / KROW, p = (at % KROW) / 16;
    return (uint32_t)((WORDS == 2 ? k & 31 : k) * ld * 2 +
                      (((p >> 1) ^ fold(k)) * 2 + (p & 1)) * 16);
  }
  // cols, WORDS 2: whether load i of wave w fetches lower words
  static __device__ __forceinline__ bool lower(int i, int w) {
    return WORDS == 2 && L == COLS && (i * NW + w) * 1024 >= 32 * KROW;
  }
  // its position in the dimension that has to be checked by hand: k for rows
  // (a row's tail is followed by the next row), r for cols
  static __device__ __forceinline__ int inner(int i, int w, int lane) {
    const int at = (i * NW + w) * 1024 + lane * 16;
    if (L == ROWS) return (((at % 128) / 16 ^ ((at / 128) & 7)) & (WORDS == 2 ? 3 : 7)) * 8;
    const int k = at / KROW, p = (at % KROW) / 16;
    return (((p >> 1) ^ fold(k)) * 2 + (p & 1)) * 8;
  }
  static __device__ __forceinline__ int fold(int k) { return (k & 3) | ((k >> 3 & 1) << 2); }

  // fragment of 16 rows from row r0 (a multiple of 16), k = 32 ks + 0..31
  static __device__ __forceinline__ v8s frag(const lchar* t, int r0, int ks, int lane) {
    const int q = lane & 15, g = lane >> 4;
    if (L == ROWS) {
      const int r = r0 + q;
      return *(const lv8s*)(t + r * 128 + ((ks * 4 + g) ^ (r & 7)) * 16);
    }
    const int k = ks * 32 + 8 * g + (q >> 2);
    const lchar* p = t + k * KROW + ((r0 >> 4) ^ fold(k)) * 32 + (q & 3) * 8;
    const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lv4s*)p);
    const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lv4s*)(p + 4 * KROW));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// Where the products' operands lie.  The second half of b[] holds the up
// projection's segments where the first holds the gate's (GATED).
struct FfnOperands {
  const void* a[FFN_MAX_SEG];
  const void* b[FFN_MAX_SEG];
  int64_t lda, ldb;
  int M, N, K;          // C's sizes (N: one projection's with GATED), k of one segment
  int nseg;
  int row0;             // the first tile's row: the others belong to another launch
  int tiles_m, tiles_n;
  int whole;            // tiles that run in one piece, the others in `splits`
  int splits;           // parts of the k steps of all segments
  __host__ __device__ int tiles() const { return tiles_m * tiles_n; }
  __host__ __device__ int groups() const { return whole + (tiles() - whole) * splits; }
};

// The place of tile `b`.  Consecutive workgroups go to different XCDs, each
// with an L2 of its own: the tiles are dealt out so that one XCD gets a
// contiguous piece of an order that walks C in bands of 8 tile rows.
__device__ __forceinline__ void tile_of(int b, int tm, int tn, int& m, int& n) {
  const int total = tm * tn, per = total / 8, rest = total % 8;
  const int x = b % 8, y = b / 8;
  const int t = x * per + (x < rest ? x : rest) + y;
  constexpr int BAND = 8;
  const int band = t / (BAND * tn), rows = min(BAND, tm - band * BAND);
  const int in = t - band * BAND * tn;
  m = band * BAND + in % rows;
  n = in / rows;
}

// GATED: B's tile rows 0 .. BN/2-1 are gate rows, the others the same columns'
// up rows; each wave's fragments are half of either.  OPS: FfnOperands, or what
// has its a[segment], b[segment], strides and sizes.  WORDS 2: every element of A and
// B is a sum of two words; a step is 32 k and three products of words (the lower ones'
// product is dropped), on four tiles where three products apart would fetch six.
template <int BM, int BN, int WM, int WN, int LA, int LB, bool F16, bool GATED,
          class OPS = FfnOperands, int WORDS = 1>
struct Gemm {
  static constexpr int NW = WM * WN, THREADS = NW * 64, BM_ = BM, BN_ = BN;
  static constexpr int FRAGS = BM / 16 * (BN / 16);   // of 16 x 16 sums
  static constexpr int MI = BM / WM / 16, NJ = BN / WN / 16;
  static constexpr int BK = FFN_BK / WORDS;   // k of a step
  using TA = Tile<LA, BM, NW, WORDS>;
  using TB = Tile<LB, BN, NW, WORDS>;
  static constexpr int LDS = 3 * TA::BYTES + 2 * TB::BYTES;
  static constexpr int COLS_N = GATED ? BN / 2 : BN;   // of C
  // WORDS 2: whether sums are put aside on the way (256 x 256 tiles have no registers
  // for that)
  static constexpr bool ASIDE = WORDS == 2 && BM == 128;
  static_assert(!GATED || LB == ROWS, "gated products have weights in rows");

  const OPS& o;
  lchar* lds;
  int wave, lane, wm, wn, m0, n0;
  uint32_t offa[TA::LOADS], offb[TB::LOADS];
  int ina[TA::LOADS], inb[TB::LOADS];

  __device__ __forceinline__ Gemm(const OPS& ops, lchar* l, int tm, int tn) : o(ops), lds(l) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    lane = threadIdx.x & 63;
    wm = wave / WN;
    wn = wave % WN;
    m0 = o.row0 + tm * BM;
    n0 = tn * COLS_N;
#pragma unroll
    for (int i = 0; i < TA::LOADS; ++i) {
      offa[i] = TA::offset(i, wave, lane, o.lda, low_a());
      ina[i] = TA::inner(i, wave, lane);
      if (LA == COLS && m0 + ina[i] >= o.M) offa[i] = OUT_OF_RANGE;
    }
#pragma unroll
    for (int i = 0; i < TB::LOADS; ++i) {
      offb[i] = TB::offset(i, wave, lane, o.ldb, low_b());
      if (GATED && up_half(i)) offb[i] -= (uint32_t)(BN / 2 * o.ldb * 2);
      inb[i] = TB::inner(i, wave, lane);
      if (LB == COLS && n0 + inb[i] >= o.N) offb[i] = OUT_OF_RANGE;
    }
  }
  // where an element's lower word lies, in elements
  __device__ __forceinline__ int low_a() const {
    if constexpr (WORDS == 2) return o.low_a;
    return 0;
  }
  __device__ __forceinline__ int low_b() const {
    if constexpr (WORDS == 2) return o.low_b;
    return 0;
  }
  __device__ __forceinline__ bool up_half(int i) const { return (i * NW + wave) * 8 >= BN / 2; }

  // C row of the first of fragment i's rows, C column of fragment j's
  __device__ __forceinline__ int frag_m(int i) const { return wm * (BM / WM) + i * 16; }
  __device__ __forceinline__ int frag_n(int j) const {   // LDS row
    if (GATED) return (j < NJ / 2 ? 0 : BN / 2) + wn * (BN / 2 / WN) + (j % (NJ / 2)) * 16;
    return wn * (BN / WN) + j * 16;
  }

  // Where an operand's next step begins and how many bytes are left of it from
  // there.  rows: up to row rows-1's k K-1; cols: up to k K-1's row rows-1.  A
  // 16-byte load that the bound cuts gives zeros whole, so the contiguous size
  // counts with the padding to 8 elements that every row of an operand has.
  struct Cursor {
    const char* at;
    int64_t left;
    __device__ v4i buffer() const { return buffer_of(at, left); }
  };
  template <int L>
  static __device__ __forceinline__ Cursor cursor(const void* p, int64_t ld, int r0, int rows, int k0, int K) {
    const char* base = (const char*)p;
    if (L == ROWS)
      return Cursor{base + ((int64_t)r0 * ld + k0) * 2,
                    ((int64_t)(rows - 1 - r0) * ld + ((K + 7) & ~7) - k0) * 2};
    return Cursor{base + ((int64_t)k0 * ld + r0) * 2,
                  ((int64_t)(K - 1 - k0) * ld + ((rows + 7) & ~7) - r0) * 2};
  }
  template <int L>
  static __device__ __forceinline__ void advance(Cursor& c, int64_t ld) {
    const int64_t step = L == ROWS ? BK * 2 : ld * BK * 2;
    c.at += step;
    c.left -= step;
  }

  // The steps that are still to be fetched, in order.
  struct Walk {
    int seg, k0;
    Cursor a, b, u;
  };
  __device__ __forceinline__ void seek(Walk& w) const {
    w.a = cursor<LA>(o.a[w.seg], o.lda, m0, o.M, w.k0, o.K);
    w.b = cursor<LB>(o.b[w.seg], o.ldb, n0, o.N, w.k0, o.K);
    if (GATED) w.u = cursor<LB>(o.b[w.seg + FFN_MAX_SEG / 2], o.ldb, n0, o.N, w.k0, o.K);
  }
  __device__ __forceinline__ void next(Walk& w) const {
    w.k0 += BK;
    if (w.k0 < o.K) {
      advance<LA>(w.a, o.lda);
      advance<LB>(w.b, o.ldb);
      if (GATED) advance<LB>(w.u, o.ldb);
    } else {
      w.k0 = 0;
      w.seg = min(w.seg + 1, o.nseg - 1);
      seek(w);
    }
  }

  // What the loads of one operand's next step need; the up rows of B's tile
  // come from a buffer of their own.
  struct Fetch {
    v4i buf, up;
    uint32_t lds;
    int k0;
  };
  // the lower words': rows have them behind the higher ones, within one buffer; those
  // of columns are a buffer of their own
  template <int L>
  static __device__ __forceinline__ v4i buffer(const Cursor& c, int low) {
    if (WORDS == 2 && L == ROWS) return buffer_of(c.at, c.left > 0 ? c.left + low * 2 : 0);
    return c.buffer();
  }
  template <int L>
  static __device__ __forceinline__ v4i lower_buffer(const Cursor& c, int low, v4i same) {
    if (WORDS == 2 && L == COLS) return buffer_of(c.at + low * 2, c.left);
    return same;
  }
  __device__ __forceinline__ Fetch fetch_a(const Walk& w, int at) const {
    const v4i b = buffer<LA>(w.a, low_a());
    return Fetch{b, lower_buffer<LA>(w.a, low_a(), b),
                 (uint32_t)(uintptr_t)(lds + at) + wave * 1024, w.k0};
  }
  __device__ __forceinline__ Fetch fetch_b(const Walk& w, int at) const {
    const v4i b = buffer<LB>(w.b, low_b());
    return Fetch{b, GATED ? w.u.buffer() : lower_buffer<LB>(w.b, low_b(), b),
                 (uint32_t)(uintptr_t)(lds + at) + wave * 1024, w.k0};
  }
  __device__ __forceinline__ void load_a(const Fetch& f, int i) const {
    load_lds(TA::lower(i, wave) ? f.up : f.buf, f.lds + i * NW * 1024,
             LA == ROWS && f.k0 + ina[i] >= o.K ? OUT_OF_RANGE : offa[i]);
  }
  __device__ __forceinline__ void load_b(const Fetch& f, int i) const {
    load_lds((GATED && up_half(i)) || TB::lower(i, wave) ? f.up : f.buf, f.lds + i * NW * 1024,
             LB == ROWS && f.k0 + inb[i] >= o.K ? OUT_OF_RANGE : offb[i]);
  }

  // Half a step: the products of the fragments a, b, row of fragments after row,
  // with the LDS reads of the next half's (na, nb: k = 32 ks .. of the tiles at
  // ta, tb) and one operand's loads of a later step dealt out between the rows.
  // A wave issues in order, so a queue of loads or reads ahead of the products
  // would idle the matrix cores until it drains.
  template <bool LOAD_A>
  __device__ __forceinline__ void half(const v8s (&a)[MI], const v8s (&b)[NJ], v4f (&acc)[MI][NJ], int ta, int tb,
                       int ks, v8s (&na)[MI], v8s (&nb)[NJ], const Fetch& f) const {
    constexpr int LOADS = LOAD_A ? TA::LOADS : TB::LOADS;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
      for (int j = i * NJ / MI; j < (i + 1) * NJ / MI; ++j)
        nb[j] = TB::frag(lds + tb, frag_n(j), ks, lane);
      na[i] = TA::frag(lds + ta, frag_m(i), ks, lane);
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = mma<F16>(b[j], a[i], acc[i][j]);
#pragma unroll
      for (int l = i * LOADS / MI; l < (i + 1) * LOADS / MI; ++l) {
        if (LOAD_A) load_a(f, l);
        else load_b(f, l);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // WORDS 2, behind half a step of the higher words' products: the products of A's
  // lower and B's higher words, with one operand's loads dealt out between the rows;
  // then those of A's higher and B's lower words, with the LDS reads of the next step's
  // higher words, each into the registers of what is not needed any more.
  __device__ __forceinline__ void lower_half(v8s (&a0)[MI], v8s (&b0)[NJ], const v8s (&a1)[MI],
                                             const v8s (&b1)[NJ], v4f (&acc)[MI][NJ], int ta, int tb,
                                             const Fetch& f) const {
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = mma<F16>(b0[j], a1[i], acc[i][j]);
#pragma unroll
      for (int l = i * TB::LOADS / MI; l < (i + 1) * TB::LOADS / MI; ++l) load_b(f, l);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
      for (int j = i * NJ / MI; j < (i + 1) * NJ / MI; ++j) b0[j] = TB::frag(lds + tb, frag_n(j), 0, lane);
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = mma<F16>(b1[j], a0[i], acc[i][j]);
      a0[i] = TA::frag(lds + ta, frag_m(i), 0, lane);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // the k steps [begin, end) of all segments' steps in order
  __device__ __forceinline__ void run(int begin, int end, v4f (&acc)[MI][NJ]) const {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    if (begin >= end) return;
    const int steps = (o.K + BK - 1) / BK;
    Walk w;
    w.seg = begin / steps;
    w.k0 = (begin % steps) * BK;
    seek(w);
    // A's tiles of this step, the next and the one after, B's of this and the next
    int a0_ = 0, a1_ = TA::BYTES, a2_ = 2 * TA::BYTES;
    int b0_ = 3 * TA::BYTES, b1_ = b0_ + TB::BYTES;
    auto fetch = [&](int at_a, int at_b) {
      const Fetch fa = fetch_a(w, at_a), fb = fetch_b(w, at_b);
#pragma unroll
      for (int l = 0; l < TA::LOADS; ++l) load_a(fa, l);
#pragma unroll
      for (int l = 0; l < TB::LOADS; ++l) load_b(fb, l);
      next(w);
    };
    fetch(a0_, b0_);
    wait_loads<0>();
    if (begin + 1 < end) fetch(a1_, b1_);
    v8s fa0[MI], fb0[NJ], fa1[MI], fb1[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) fb0[j] = TB::frag(lds + b0_, frag_n(j), 0, lane);
#pragma unroll
    for (int i = 0; i < MI; ++i) fa0[i] = TA::frag(lds + a0_, frag_m(i), 0, lane);
    v4f aside[ASIDE ? MI : 1][ASIDE ? NJ : 1] = {};
    const int apart = end - begin <= 8 ? 0 : 7;
    for (int s = begin; s < end; ++s) {
      // behind the last step there is nothing to load: empty buffers
      if (s + 2 >= end) w.a.left = w.b.left = w.u.left = 0;
      const Fetch fa = fetch_a(w, a2_), fb = fetch_b(w, b0_);
      __builtin_amdgcn_sched_barrier(0);
      half<true>(fa0, fb0, acc, a0_, b0_, 1, fa1, fb1, fa);
      // all but A's tile of the step after the next one has arrived, and nobody
      // reads this step's tiles any more
      wait_loads<TA::LOADS>();
      __builtin_amdgcn_sched_barrier(0);
      // The matrix cores add a product's 32 terms to a sum with about twice the error of
      // one addition in fp32, at random: sums of positive terms are 8.5e-8 off after 8
      // products (root mean square), 2.4e-7 after 64, 6.3e-7 after 448.  Three products a
      // step do so at the whole sum's size.  So the sums are added up outside of them
      // every eight steps, or at every one of a few, and before the lower words'
      // products, which then start from nothing.  (Orthogonalised in fp32,
      // 4067 x 2773 was 2.2e-6 off and is 0.8e-6, 34 x 3558 2.5e-6 and 1.8e-6, in the
      // same time.  At every second step 24 matrices of up to 333 rows take 3% longer;
      // dealt out between the products at every step, spills and twice the time.)
      if constexpr (ASIDE)
        if (((s - begin) & apart) == 0) {
#pragma unroll
          for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
              aside[i][j] += acc[i][j];
              acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
            }
          __builtin_amdgcn_sched_barrier(0);
        }
      // (after the last step the reads are of no use, within LDS)
      if constexpr (WORDS == 2) lower_half(fa0, fb0, fa1, fb1, acc, a1_, b1_, fb);
      else half<false>(fa1, fb1, acc, a1_, b1_, 0, fa0, fb0, fb);
      next(w);
      const int a = a0_, b = b0_;
      a0_ = a1_;
      a1_ = a2_;
      a2_ = a;
      b0_ = b1_;
      b1_ = b;
    }
    if constexpr (ASIDE)
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] += aside[i][j];
    wait_loads<0>();   // LDS belongs to the next workgroup once this one has ended
  }
};

}  // namespace scao
