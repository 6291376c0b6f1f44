// The kernels of the Newton-Schulz orthogonalisation.
//
//   X = G / (|G| + eps), then for every step, on the smaller side of X:
//   A = X X^T, B = a + b A + c A A, X <- B X      (wide: rows <= cols)
//   A = X^T X, B = a + b A + c A A, X <- X B      (tall)
//
// Nothing is transposed in memory: the tiled product reads an operand with k or
// with its rows contiguous.  A and B are symmetric, so only the tiles on and below
// the diagonal are computed and the others stored as their mirror image.
//
// Words of the products.  X, A and B are fp16 or, P = 2, a sum of two fp16 words (22
// significant bits, multiplied as three products of words), a group's choice; scaled by
// powers of two that the host chooses from what the polynomial can reach, so that
// neither end of fp16's range matters: |X|, |A| and |B| are bounded by their largest
// singular value.  fp16 has three bits more than bf16 at the same rate; each of the
// three is rounded once a step, which leaves results of 640 x 640 1.2e-3 off (five
// steps; 4096 x 1024 0.8e-3, 2048 x 512 1.4e-3), a bf16 result's own rounding 1.7e-3.  Sums and b A are fp32.  a is part of B:
// a X beside the product is no more exact (1.3e-3), and would read X once more at every
// tile's end, when all of the chip does (3.6% of the time).
//
// What bounds it: the chip's power in long updates (14336 x 4096: matrix cores busy 66%
// of the cycles at 1.85 GHz, 378 us an update, 1.27 PFLOP/s); the count of tiles in the
// symmetric products (136 of 256 x 256 on 256 CUs; 528 of 128 x 128, the 16 behind the
// last round in 16 parts: 86 us for 4096 x 4096 with their join, 271 for the Gram matrix
// over 14336); launches for small matrices, about 5 us each whatever they hold.
//
// All matrices of a call go through the same launches, whatever their shapes: a
// launch's tiles are those of up to ORTHO_GROUPS groups of one shape each, the ones
// with the longest sums first.
#pragma once

#include "ffn_kernels.hpp"

namespace scao {

constexpr int ORTHO_GROUPS = 16;     // shapes a pass
constexpr int ORTHO_MATRICES = 64;   // matrices a pass
constexpr int ORTHO_PARTS = 1024;    // sums of squares a matrix

enum { ORTHO_GRAM, ORTHO_SQUARE, ORTHO_UPDATE };
// where an update goes: the next X, the result, or (the optimiser) the parameter
enum { ORTHO_NEXT, ORTHO_RESULT, ORTHO_PARAMETER };

// Matrices of one shape, with their buffers in the workspace one after the other.
struct OrthoGroup {
  int64_t x, y, a, b;        // bytes from the workspace's start: X, the next X, A, B
  int64_t x_step, a_step;    // bytes from a matrix's X to the next one's; of A and B
  int rows, cols, ldx, lda;
  int first, count;          // entries of the pass's tables
  int words;                 // 1 or 2
  int per, tiles_m, tiles_n; // tiles of a matrix
  int tile0;                 // tiles of the groups before
};
// A phase's tiles in order.  The first `whole` go one to a workgroup, the others' k
// steps in `splits` parts.  (Parts of one length for every tile, and not shares of
// all steps wherever a tile ends: those balance 136 tiles on 256 CUs, but then no two
// workgroups of an XCD read the same k at a time, and its L2 serves nobody: 14336 x
// 4096's Gram matrix 269 us, with three parts a tile 251.)
struct OrthoPhase {
  OrthoGroup g[ORTHO_GROUPS];
  char* base;
  float* partial;            // parts of split tiles
  int groups, tiles, whole, splits;
  float by, keep, diagonal;  // of the product; of A; added to B's diagonal
};
struct OrthoOut {
  void* p[ORTHO_MATRICES];
  int ld[ORTHO_MATRICES];
  float rate[ORTHO_MATRICES], decay[ORTHO_MATRICES];   // p <- decay p - rate update
  uint8_t dt[ORTHO_MATRICES];
};

// What the tiled product needs of one of this group's products: one segment, and where
// an element's lower word lies.
struct OrthoWords {
  const char* p;
  __device__ __forceinline__ const void* operator[](int) const { return p; }
};
struct OrthoOperands {
  OrthoWords a, b;
  int64_t lda, ldb;
  int low_a, low_b;
  int M, N, K, nseg, row0;
};
// ld: elements of a row of one word; the rows of both words take turns
template <int P>
__device__ __forceinline__ OrthoOperands ortho_operands(const char* a, int lda, const char* b,
                                                        int ldb, int M, int N, int K) {
  return OrthoOperands{{a}, {b}, (int64_t)P * lda, (int64_t)P * ldb, lda, ldb, M, N, K, 1, 0};
}

// four values as fp16 words: rounded, or with the rest in a second word
template <int P>
__device__ __forceinline__ void ortho_words(v4f x, v2u (&w)[P]) {
  w[0] = v4f_to_halves(SCAO_F16, x);
  if constexpr (P == 2) w[1] = v4f_to_halves(SCAO_F16, x - halves_to_v4f(SCAO_F16, w[0]));
}

// ---------------------------------------------------------- products -------
// The tile of place t of a group's tiles.  As tile_of does it, one XCD gets a
// contiguous piece of them.
__device__ __forceinline__ void ortho_tile_of(const OrthoGroup& g, bool lower, int t, int& matrix,
                                              int& tm, int& tn) {
  const int total = g.count * g.per, each = total / 8, rest = total % 8;
  const int x = t % 8, at = x * each + (x < rest ? x : rest) + t / 8;
  matrix = at / g.per;
  const int in = at - matrix * g.per;
  if (lower) {   // row tm's tiles 0 .. tm behind those of the rows before
    tm = (int)((sqrtf(8.f * in + 1.f) - 1.f) * 0.5f);
    if (tm * (tm + 1) / 2 > in) --tm;
    if ((tm + 1) * (tm + 2) / 2 <= in) ++tm;
    tn = in - tm * (tm + 1) / 2;
    return;
  }
  constexpr int BAND = 8;
  const int band = in / (BAND * g.tiles_n), rows = min(BAND, g.tiles_m - band * BAND);
  const int rem = in - band * BAND * g.tiles_n;
  tm = band * BAND + rem % rows;
  tn = rem / rows;
}
__device__ __forceinline__ int ortho_group_of(const OrthoPhase& ph, int tile) {
  int k = 0;
  for (int i = 1; i < ph.groups; ++i)
    if (tile >= ph.g[i].tile0) k = i;
  return k;
}
// where the phase's product is stored, and what is added to it
struct OrthoTarget {
  uint16_t* to;
  const uint16_t* add;
  int plane, M, N, cols;   // from one word's row to the next's; cols: N rounded up to 8
  int64_t ld;
  bool mirror;             // a tile below the diagonal
};
template <int PHASE>
__device__ __forceinline__ OrthoTarget ortho_target(const OrthoPhase& ph, const OrthoGroup& g,
                                                    int matrix, bool mirror) {
  char* x = ph.base + matrix * g.x_step;
  char* a = ph.base + matrix * g.a_step;
  OrthoTarget t;
  t.mirror = PHASE != ORTHO_UPDATE && mirror;
  if (PHASE == ORTHO_UPDATE) {
    t.to = (uint16_t*)(x + g.y);
    t.add = nullptr;
    t.plane = g.ldx;
    t.M = g.rows;
    t.N = g.cols;
  } else {
    t.to = (uint16_t*)(a + (PHASE == ORTHO_GRAM ? g.a : g.b));
    t.add = (const uint16_t*)(a + g.a);
    t.M = t.N = min(g.rows, g.cols);
    t.plane = g.lda;
  }
  t.ld = (int64_t)g.words * t.plane;
  t.cols = (t.N + 7) & ~7;
  return t;
}

// the inverse of join_pair
__device__ __forceinline__ void part_pair(v4u_t w, v2u& p, v2u& q) {
  const auto a = __builtin_amdgcn_permlane16_swap(w[0], w[2], false, false);
  const auto b = __builtin_amdgcn_permlane16_swap(w[1], w[3], false, false);
  p = v2u{a[0], b[0]};
  q = v2u{a[1], b[1]};
}
// Four lanes next to each other hold four columns of a row each; each gets one of
// these columns' four rows instead.
__device__ __forceinline__ v2u turn4(v2u w, int lane) {
  const uint32_t sel = lane & 1 ? 0x03020706u : 0x05040100u;
  uint32_t n[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    n[i] = __builtin_amdgcn_perm(__builtin_amdgcn_mov_dpp((int)w[i], 0xB1, 15, 15, true), w[i], sel);
  const bool up = lane & 2;
  const uint32_t own = up ? n[1] : n[0];
  const uint32_t other = __builtin_amdgcn_mov_dpp((int)(up ? n[0] : n[1]), 0x4E, 15, 15, true);
  return up ? v2u{other, own} : v2u{own, other};
}

// Two fragments next to each other, the first at row m (this lane's) and column n.
template <int P, int PHASE>
struct OrthoPair {
  v4u_t w[P];
  __device__ __forceinline__ void load(const OrthoTarget& t, int m, int n, int lane) {
    if (PHASE != ORTHO_SQUARE) return;
    n += pair_column(lane);
    const bool in = m < t.M && n < t.cols;
#pragma unroll
    for (int i = 0; i < P; ++i)
      w[i] = in ? (v4u_t) * (const gv4u_a16*)(t.add + m * t.ld + n + i * t.plane)
                : v4u_t{0, 0, 0, 0};
  }
  // by c, of a square by c + keep A + diagonal, likewise d
  __device__ __forceinline__ void sum(const OrthoPhase& ph, int m, int n, int lane, v4f& c,
                                      v4f& d) const {
    c *= ph.by;
    d *= ph.by;
    if (PHASE != ORTHO_SQUARE) return;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      v2u p, q;
      part_pair(w[i], p, q);
      const v4f x = halves_to_v4f(SCAO_F16, p), y = halves_to_v4f(SCAO_F16, q);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        c[t] = fmaf(ph.keep, x[t], c[t]);
        d[t] = fmaf(ph.keep, y[t], d[t]);
      }
    }
    n += 4 * (lane >> 4);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (n + t == m) c[t] += ph.diagonal;
      if (n + 16 + t == m) d[t] += ph.diagonal;
    }
  }
};

// A tile's mirror image goes through LDS, which the products need no more: rows of
// 16-byte stores.  (Stored from the registers, 32 bytes of a row at a time, it took 8 us
// of a 256 x 256 tile's 16 beside its k steps, 16 of 26 with two words.)  Rows of BM
// elements and 32 bytes, so that the 16 lanes that write four rows each meet all banks.
template <int BM>
struct OrthoImage {
  static constexpr int ROW = BM * 2 + 32;
  static constexpr int BYTES = BM * ROW;
  typedef __attribute__((address_space(3))) v2u lv2u;
  typedef __attribute__((address_space(3))) v4u_t lv4u;
  // a fragment's words, from row m and column n of the tile
  static __device__ __forceinline__ void put(lchar* lds, int m, int n, int lane, v2u w) {
    const int q = lane & 3;
    *(lv2u*)(lds + (n + 4 * (lane >> 4) + q) * ROW + (m + (lane & 15) - q) * 2) = turn4(w, lane);
  }
  // plane `to` of the matrix; row0, col0: the image's place
  static __device__ __forceinline__ void store(const lchar* lds, const OrthoTarget& t, uint16_t* to,
                                               int row0, int col0) {
    constexpr int PIECES = BM / 8, THREADS = BM * 2;
#pragma unroll 4
    for (int i = 0; i < BM * PIECES / THREADS; ++i) {
      const int at = i * THREADS + threadIdx.x, r = at / PIECES, c = at % PIECES * 8;
      if (col0 + c < t.cols)
        *(gv4u_a16*)(to + (row0 + r) * t.ld + col0 + c) = *(const lv4u*)(lds + r * ROW + c * 2);
    }
  }
};

// mirror: the image too, 32 bytes of a row at a time
template <int P>
__device__ __forceinline__ void ortho_store(const OrthoTarget& t, bool mirror, int m, int n, int lane,
                                            v4f c, v4f d) {
  v2u p[P], q[P];
  ortho_words<P>(c, p);
  ortho_words<P>(d, q);
  const int at = n + pair_column(lane);
  const bool in = m < t.M && at < t.cols;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const v4u_t w = join_pair(p[i], q[i]);
    if (in) *(gv4u_a16*)(t.to + m * t.ld + at + i * t.plane) = w;
  }
  if (!mirror) return;
  // (a row of C is a column of the image, so C's padding rows are stored as the
  // image's padding columns; a tile below the diagonal has no padding columns)
  const int dm = lane & 15, row = n + 4 * (lane >> 4) + (dm & 3), col = m - (dm & 3);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const v2u a = turn4(p[i], lane), b = turn4(q[i], lane);
    if (col < t.cols) {
      uint16_t* to = t.to + row * t.ld + col + i * t.plane;
      typedef __attribute__((address_space(1))) v2u gv2u_a8;
      *(gv2u_a8*)to = a;
      *(gv2u_a8*)(to + 16 * t.ld) = b;
    }
  }
}

// the last update: four columns from n of row m, in the type and place of the result
struct OrthoPlace {
  void* p;
  int ld, dt;
  float rate, decay;
};
template <int DEST>
__device__ __forceinline__ void ortho_put4(const OrthoPlace& o, const OrthoTarget& t, int m, int n,
                                           v4f c) {
  const int left = t.N - n;
  if (m >= t.M || left <= 0) return;
  const int64_t at = (int64_t)m * o.ld + n;
  const int mask = left >= 4 ? 15 : (1 << left) - 1;
  if (DEST == ORTHO_PARAMETER) {
    const v4f p = ld4(o.p, SCAO_F32, at, left >= 4, mask);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = fmaf(-o.rate, c[i], o.decay * p[i]);
  }
  st4(o.p, SCAO_F32, at, c, left >= 4, mask);
}
template <int DEST>
__device__ __forceinline__ void ortho_put(const OrthoPlace& o, const OrthoTarget& t, int m, int n,
                                          int lane, v4f c, v4f d) {
  const int dt = o.dt;
  if (dt == SCAO_F32) {
    n += 4 * (lane >> 4);
    ortho_put4<DEST>(o, t, m, n, c);
    ortho_put4<DEST>(o, t, m, n + 16, d);
    return;
  }
  const int at = n + pair_column(lane);
  uint16_t* to = (uint16_t*)o.p + (int64_t)m * o.ld + at;
  const bool in = m < t.M && at < t.N, full = in && at + 8 <= t.N;
  if (DEST == ORTHO_PARAMETER) {
    v4u_t w = {0, 0, 0, 0};
    if (full) {
      w = *(const gv4u_a2*)to;
    } else if (in) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at + i < t.N) w[i / 2] |= (uint32_t)((const gu16*)to)[i] << (16 * (i & 1));
    }
    v2u p, q;
    part_pair(w, p, q);
    const v4f x = halves_to_v4f(dt, p), y = halves_to_v4f(dt, q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = fmaf(-o.rate, c[i], o.decay * x[i]);
      d[i] = fmaf(-o.rate, d[i], o.decay * y[i]);
    }
  }
  v2u p, q;
  if (dt == SCAO_BF16) {
    p = v2u{pk_bf16(c[0], c[1]), pk_bf16(c[2], c[3])};
    q = v2u{pk_bf16(d[0], d[1]), pk_bf16(d[2], d[3])};
  } else {
    p = v4f_to_halves(SCAO_F16, c);
    q = v4f_to_halves(SCAO_F16, d);
  }
  const v4u_t w = join_pair(p, q);
  if (full) {
    *(gv4u_a2*)to = w;
  } else if (in) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at + i < t.N) ((gu16*)to)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
  }
}

template <int P, int PHASE, int DEST>
__device__ __forceinline__ void ortho_finish(const OrthoPhase& ph, const OrthoPlace& o,
                                             const OrthoTarget& t, const OrthoPair<P, PHASE>& add,
                                             bool mirror, int m, int n, int lane, v4f& c, v4f& d) {
  add.sum(ph, m, n, lane, c, d);
  if constexpr (DEST == ORTHO_NEXT) ortho_store<P>(t, mirror, m, n, lane, c, d);
  else ortho_put<DEST>(o, t, m, n, lane, c, d);
}
template <int DEST>
__device__ __forceinline__ OrthoPlace ortho_place(const OrthoOut& o, int e) {
  if (DEST == ORTHO_NEXT) return OrthoPlace{};
  return OrthoPlace{o.p[e], o.ld[e], o.dt[e], o.rate[e], o.decay[e]};
}

template <int P, int BM, int LA, int LB>
using OrthoGemm = Gemm<BM, BM, 2, BM == 256 ? 4 : 2, LA, LB, true, false, OrthoOperands, P>;

template <class G, int P, int PHASE, int DEST>
__device__ __forceinline__ void ortho_tile(char* smem, const OrthoPhase& ph, const OrthoOut& out,
                                           const OrthoGroup& g, const OrthoOperands& o, int matrix,
                                           int tm, int tn, int tile, int part) {
  G gm(o, (lchar*)smem, tm, tn);
  const int steps = (o.K + G::BK - 1) / G::BK;
  const bool split = part >= 0;
  const int per = split ? (steps + ph.splits - 1) / ph.splits : steps;
  const int begin = split ? part * per : 0;
  v4f acc[G::MI][G::NJ];
  gm.run(begin, min(steps, begin + per), acc);
  const int lane = gm.lane;
  if (split) {
    gv4f_a16* to = (gv4f_a16*)ph.partial +
                   ((int64_t)part * (ph.tiles - ph.whole) + (tile - ph.whole)) * (G::FRAGS * 64) +
                   lane;
#pragma unroll
    for (int i = 0; i < G::MI; ++i)
#pragma unroll
      for (int j = 0; j < G::NJ; ++j)
        to[(gm.frag_m(i) / 16 * (G::BN_ / 16) + gm.frag_n(j) / 16) * 64] = acc[i][j];
    return;
  }
  const OrthoTarget t = ortho_target<PHASE>(ph, g, matrix, tm > tn);
  const OrthoPlace to = ortho_place<DEST>(out, g.first + matrix);
  // what is added is loaded for several rows of fragments at a time, as a wait for
  // loads also waits for the stores before them
  constexpr int BATCH = G::MI / P / (G::MI > 4 ? 2 : 1);
#pragma unroll
  for (int i0 = 0; i0 < G::MI; i0 += BATCH) {
    OrthoPair<P, PHASE> add[BATCH][G::NJ / 2];
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
#pragma unroll
      for (int j = 0; j < G::NJ; j += 2)
        add[i][j / 2].load(t, gm.m0 + gm.frag_m(i0 + i) + (lane & 15), gm.n0 + gm.frag_n(j), lane);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
#pragma unroll
      for (int j = 0; j < G::NJ; j += 2)
        ortho_finish<P, PHASE, DEST>(ph, to, t, add[i][j / 2], false,
                                     gm.m0 + gm.frag_m(i0 + i) + (lane & 15), gm.n0 + gm.frag_n(j),
                                     lane, acc[i0 + i][j], acc[i0 + i][j + 1]);
    __builtin_amdgcn_sched_barrier(0);
  }
  if constexpr (PHASE != ORTHO_UPDATE) {
    if (!t.mirror) return;
    using Image = OrthoImage<G::BM_>;
    static_assert(Image::BYTES <= G::LDS, "the image fits");
    // (the last of run() was a barrier: nobody reads the products' tiles any more.  The
    // lane is hidden from the compiler, which would keep the addresses that follow from
    // it in registers from before the products on: there are none to spare.)
    int at = lane;
    asm volatile("" : "+v"(at));
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (p) __syncthreads();
#pragma unroll
      for (int i = 0; i < G::MI; ++i)
#pragma unroll
        for (int j = 0; j < G::NJ; ++j) {
          v2u w[P];
          ortho_words<P>(acc[i][j], w);
          Image::put((lchar*)smem, gm.frag_m(i), gm.frag_n(j), at, w[p]);
          __builtin_amdgcn_sched_barrier(0);
        }
      __syncthreads();
      Image::store((const lchar*)smem, t, t.to + p * t.plane, gm.n0, gm.m0);
    }
  }
}

template <int P, int BM, int PHASE, int DEST>
__device__ __forceinline__ void ortho_product(char* smem, const OrthoPhase& ph, const OrthoOut& out,
                                              const OrthoGroup& g, int matrix, int tm, int tn,
                                              int tile, int part) {
  using RR = OrthoGemm<P, BM, ROWS, ROWS>;
  using RC = OrthoGemm<P, BM, ROWS, COLS>;
  using CC = OrthoGemm<P, BM, COLS, COLS>;
  const char* x = ph.base + matrix * g.x_step + g.x;
  const char* a = ph.base + matrix * g.a_step + (PHASE == ORTHO_SQUARE ? g.a : g.b);
  const bool wide = g.rows <= g.cols;
  const int s = wide ? g.rows : g.cols;
  if constexpr (PHASE == ORTHO_SQUARE) {
    const OrthoOperands o = ortho_operands<P>(a, g.lda, a, g.lda, s, s, s);
    ortho_tile<RR, P, PHASE, DEST>(smem, ph, out, g, o, matrix, tm, tn, tile, part);
  } else if constexpr (PHASE == ORTHO_GRAM) {
    const OrthoOperands o =
        ortho_operands<P>(x, g.ldx, x, g.ldx, s, s, wide ? g.cols : g.rows);
    if (wide) ortho_tile<RR, P, PHASE, DEST>(smem, ph, out, g, o, matrix, tm, tn, tile, part);
    else ortho_tile<CC, P, PHASE, DEST>(smem, ph, out, g, o, matrix, tm, tn, tile, part);
  } else if (wide) {
    const OrthoOperands o = ortho_operands<P>(a, g.lda, x, g.ldx, g.rows, g.cols, s);
    ortho_tile<RC, P, PHASE, DEST>(smem, ph, out, g, o, matrix, tm, tn, tile, part);
  } else {
    const OrthoOperands o = ortho_operands<P>(x, g.ldx, a, g.lda, g.rows, g.cols, s);
    ortho_tile<RR, P, PHASE, DEST>(smem, ph, out, g, o, matrix, tm, tn, tile, part);
  }
}
template <int BM, int PHASE, int DEST>
__global__ __launch_bounds__(BM * 2, 2) void k_ortho(const OrthoPhase ph, const OrthoOut out) {
  using G = OrthoGemm<1, BM, ROWS, ROWS>;
  static_assert(G::THREADS == BM * 2, "a wave for every 32 rows");
  __shared__ __attribute__((aligned(1024))) char smem[G::LDS];
  const int b = blockIdx.x, rest = ph.tiles - ph.whole;
  const int part = b < ph.whole ? -1 : (b - ph.whole) / rest;
  const int tile = part < 0 ? b : ph.whole + (b - ph.whole) % rest;
  const OrthoGroup& g = ph.g[ortho_group_of(ph, tile)];
  int matrix, tm, tn;
  ortho_tile_of(g, PHASE != ORTHO_UPDATE, tile - g.tile0, matrix, tm, tn);
  if (g.words == 2) ortho_product<2, BM, PHASE, DEST>(smem, ph, out, g, matrix, tm, tn, tile, part);
  else ortho_product<1, BM, PHASE, DEST>(smem, ph, out, g, matrix, tm, tn, tile, part);
}

// The parts of split tiles, added in order: a wave takes two fragments.
template <int P>
struct OrthoWordCount {
  static constexpr int value = P;
};
template <int BM, int PHASE, int DEST>
__global__ __launch_bounds__(256) void k_ortho_join(const OrthoPhase ph, const OrthoOut out) {
  constexpr int F = BM / 16, PAIRS = F * F / 2;   // of a tile
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int rest = ph.tiles - ph.whole, lane = threadIdx.x & 63;
  if (at >= (int64_t)rest * PAIRS) return;
  const int tile = ph.whole + (int)(at / PAIRS), in = (int)(at % PAIRS);
  const OrthoGroup& g = ph.g[ortho_group_of(ph, tile)];
  int matrix, tm, tn;
  ortho_tile_of(g, PHASE != ORTHO_UPDATE, tile - g.tile0, matrix, tm, tn);
  const OrthoTarget t = ortho_target<PHASE>(ph, g, matrix, tm > tn);
  const int fm = in / (F / 2), fn = in % (F / 2) * 2;
  const int m = tm * BM + fm * 16 + (lane & 15), n = tn * BM + fn * 16;
  // (whole fragments outside; the mirror image's padding columns are C's rows)
  if (tm * BM + fm * 16 >= ((t.M + 7) & ~7) || n >= t.cols) return;
  const gv4f_a16* p = (const gv4f_a16*)ph.partial +
                      ((int64_t)(tile - ph.whole) * F * F + fm * F + fn) * 64 + lane;
  const int64_t all = (int64_t)rest * F * F * 64;
  v4f c = {0.f, 0.f, 0.f, 0.f}, d = c;
  constexpr int BATCH = 4;
  for (int s = 0; s < ph.splits; s += BATCH) {
    v4f pc[BATCH], pd[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (s + i < ph.splits) {
        pc[i] = p[(s + i) * all];
        pd[i] = p[(s + i) * all + 64];
      }
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (s + i < ph.splits) {
        c += pc[i];
        d += pd[i];
      }
  }
  const OrthoPlace to = ortho_place<DEST>(out, g.first + matrix);
  auto finish = [&](auto words) {
    constexpr int P = decltype(words)::value;
    OrthoPair<P, PHASE> add;
    add.load(t, m, n, lane);
    ortho_finish<P, PHASE, DEST>(ph, to, t, add, t.mirror, m, n, lane, c, d);
  };
  if (g.words == 2) finish(OrthoWordCount<2>{});
  else finish(OrthoWordCount<1>{});
}

// --------------------------------------------------------- launches --------
template <int BM, int PHASE, int DEST>
void ortho_launch(const OrthoPhase& ph, const OrthoOut& out, hipStream_t st) {
  const int rest = ph.tiles - ph.whole;
  k_ortho<BM, PHASE, DEST><<<ph.whole + rest * ph.splits, BM * 2, 0, st>>>(ph, out);
  if (rest)
    k_ortho_join<BM, PHASE, DEST>
        <<<(int)(((int64_t)rest * (BM / 16) * (BM / 16) / 2 + 3) / 4), 256, 0, st>>>(ph, out);
}
template <int BM>
void ortho_launch(int phase, int dest, const OrthoPhase& ph, const OrthoOut& out, hipStream_t st) {
  if (phase == ORTHO_GRAM) ortho_launch<BM, ORTHO_GRAM, ORTHO_NEXT>(ph, out, st);
  else if (phase == ORTHO_SQUARE) ortho_launch<BM, ORTHO_SQUARE, ORTHO_NEXT>(ph, out, st);
  else if (dest == ORTHO_NEXT) ortho_launch<BM, ORTHO_UPDATE, ORTHO_NEXT>(ph, out, st);
  else if (dest == ORTHO_RESULT) ortho_launch<BM, ORTHO_UPDATE, ORTHO_RESULT>(ph, out, st);
  else ortho_launch<BM, ORTHO_UPDATE, ORTHO_PARAMETER>(ph, out, st);
}
// instantiated in ortho_tiles128.hip and ortho_tiles256.hip
void ortho_tiles128(int phase, int dest, const OrthoPhase& ph, const OrthoOut& out, hipStream_t st);
void ortho_tiles256(int phase, int dest, const OrthoPhase& ph, const OrthoOut& out, hipStream_t st);

}  // namespace scao
