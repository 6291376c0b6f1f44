// A step of matrices of a few hundred rows in one launch.
//
//   A X, (A X) X^T and ((A X) X^T) X = A A X need 16 rows of X and all of X, but no
//   other rows of A: a workgroup takes a panel of 16 rows through four products,
//
//     A' = X' X^T,  Y = A' X,  A'' = Y X^T (= (A A)'),  Z = A'' X,
//     X' <- a X' + b Y + c Z,
//
// with X read from L2 and the panel in LDS.  That is twice the operations of the
// products of whole matrices, and one launch instead of three.
//
// X is kept in both orders, its rows for the products with X^T and its columns for
// those with X, and as the matrix cores take it: pieces of 16 rows by 32 k, 8 k of row
// lane % 16 from 8 (lane / 16) on a lane, 1 KB a word in a row.  A wave's load is one
// such piece, and none of X is read twice in a product (as rows, 16 pieces of 64 bytes
// a load, a step of 256 x 256 took 22 us).  Zeros up to 32 rows and columns.
//
// Sums, b Y and a X' are fp32.  A' and A'' are rounded to two words whatever the group's
// are, as an error of theirs reaches all that follows from them: with one word each,
// results of 256 x 256 were 1.5e-3 off after the published five steps and those of 256 x
// 1024 1.9e-3, where tiles leave 1.3e-3 and 1.1e-3; with two they are 1.0e-3 and 0.7e-3
// off, in the time of one (256 x 256 59 us, 384 x 384 106 for 101).  X, and Y beside A' X,
// have the group's words.
//
// What bounds it: reads of X from L2, 7.5 to 15 us a MB and panel, and about 0.8 us a
// product until its first sums.  Five steps of 256 x 256 in one word: 59 us, of which
// the launches alone are 25 (tiles 125; 16 matrices 82 and 129, 64 240 and 151); of two
// words 86 (162); 384 x 384 106 (145), 512 x 512 152 (161), 256 x 1024 177 (138).  The
// host takes whichever its estimates say.  With one word and up to 256 columns a wave's
// pieces of X, in either order, stay in its registers for the step: 70 to 63 us of 256 x
// 256.  The first pieces of a product fetched before the barrier ahead of it spill:
// slower in every other case (512 x 512: 156 to 184).
#pragma once

#include "ortho_small.hpp"

namespace scao {

constexpr int PANEL = 16;
constexpr int PANEL_THREADS = 1024, PANEL_WAVES = PANEL_THREADS / 64;
constexpr int PANEL_SIDE = 512, PANEL_LENGTH = 1024;   // of s, of l
constexpr int PANEL_BLOCKS = PANEL_LENGTH / 16 / PANEL_WAVES;   // a wave's blocks of l
constexpr int PANEL_LDS = 156 * 1024;

// Matrices of one shape: X as s rows of l and as l rows of s, all of them multiples of 32
// with the zeros behind.
struct PanelGroup {
  int64_t rows, columns, next_rows, next_columns;   // bytes from the workspace's start
  int s, l, source_s, source_l;
  int first, count, words, wide;
  int per, block0;                                  // panels a matrix; of the groups before
  int parts;                                        // sums of squares a matrix
};
__host__ __device__ inline int panel_bytes(const PanelGroup& g) { return g.words * g.s * g.l * 2; }
struct OrthoPanels {
  PanelGroup g[ORTHO_GROUPS];
  char* base;
  int groups;
  float gram, second, third;        // of A', Y and A'' when they become words (A's two)
  float a, b, c;                    // of X's words, of Y's and of Z's sums
};
static_assert(sizeof(OrthoPanels) + sizeof(OrthoOut) <= 4096, "kernel arguments are limited to 4 KiB");

// (panels of A and A A have two words whatever X has)
__host__ __device__ inline int panel_lds(const PanelGroup& g) {
  return PANEL * 2 * (g.words * 2 * g.l + 2 * g.s);
}
// whether a wave's 128 registers hold its pieces of X in either order
__host__ __device__ inline bool panel_held(const PanelGroup& g) { return g.words == 1 && g.l <= 256; }
typedef __attribute__((address_space(1))) v8s gv8s;
typedef __attribute__((address_space(3))) v4u_t lv4u;

__device__ __forceinline__ const PanelGroup& panel_group(const PanelGroup* g, int groups, int& in) {
  int k = 0;
  for (int i = 1; i < groups; ++i)
    if ((int)blockIdx.x >= g[i].block0) k = i;
  in = blockIdx.x - g[k].block0;
  return g[k];
}

// Rows j .. j + 15 of a matrix in memory times the panel's, over k: what this lane holds
// is of panel row lane % 16 and of rows j + 4 (lane / 16) .. + 3.  The next pieces are
// under way during the products of some.  The panel has W words an element, the matrix P.
template <int P, int W>
struct PanelRows {
  static constexpr int STEPS = P == 1 ? 8 : 4;
  typedef v8s Pieces[STEPS][P];
  Pieces first;
  const char* at;
  int pieces;

  __device__ __forceinline__ void fetch(int k0, Pieces& w) const {
#pragma unroll
    for (int h = 0; h < STEPS; ++h)
      if (k0 + h < pieces)
#pragma unroll
        for (int i = 0; i < P; ++i) w[h][i] = *(const gv8s*)(at + ((k0 + h) * P + i) * 1024);
  }
  __device__ __forceinline__ void begin(const char* x, int j, int k_end, int lane) {
    pieces = k_end / 32;
    at = x + (int64_t)(j / 16) * pieces * P * 1024 + lane * 16;
    fetch(0, first);
  }
  __device__ __forceinline__ void add(const lchar* panel, int lane, int k0, const Pieces& w,
                                      v4f (&c)[3]) const {
#pragma unroll
    for (int h = 0; h < STEPS; ++h)
      if (k0 + h < pieces) {
        const lchar* t = panel + (k0 + h) * W * 1024 + lane * 16;
        const v8s hi = *(const lv8s*)t;
        if constexpr (W == 1) {
          c[h & 1] = mma<true>(w[h][0], hi, c[h & 1]);
        } else {
          const v8s lo = *(const lv8s*)(t + 1024);
          if constexpr (P == 2) c[2] = mma<true>(w[h][1], hi, c[2]);
          c[0] = mma<true>(w[h][0], lo, c[0]);
          c[1] = mma<true>(w[h][0], hi, c[1]);
        }
      }
  }
  // of all pieces, which `first` holds and goes on holding
  __device__ __forceinline__ v4f product(const lchar* panel, int lane) const {
    v4f c[3] = {};
    add(panel, lane, 0, first, c);
    return sum(c);
  }
  static __device__ __forceinline__ v4f sum(const v4f (&c)[3]) {
    return P == 1 ? c[0] + c[1] : (c[2] + c[0]) + c[1];
  }
};
template <int P, int W>
__device__ __forceinline__ v4f panel_product(const char* x, int j, int k_end, const lchar* panel,
                                             int lane) {
  PanelRows<P, W> r;
  typename PanelRows<P, W>::Pieces next;
  r.begin(x, j, k_end, lane);
  v4f c[3] = {};
  for (int k = 0; k < r.pieces; k += 2 * r.STEPS) {
    r.fetch(k + r.STEPS, next);
    r.add(panel, lane, k, r.first, c);
    r.fetch(k + 2 * r.STEPS, r.first);
    r.add(panel, lane, k + r.STEPS, next, c);
  }
  return r.sum(c);
}

// where k = n of row m (of 16) lies in a panel, in bytes
template <int P>
__device__ __forceinline__ int panel_at(int m, int n) {
  return n / 32 * P * 1024 + (m + 16 * (n % 32 / 8)) * 16 + n % 8 * 2;
}
// columns n .. n + 3 of the panel's row m
template <int P>
__device__ __forceinline__ void panel_put(lchar* t, int m, int n, v4f c) {
  v2u w[P];
  ortho_words<P>(c, w);
#pragma unroll
  for (int i = 0; i < P; ++i) *(lv2u*)(t + panel_at<P>(m, n) + i * 1024) = w[i];
}

// ALL: a wave has one block of columns in either product, whose pieces it keeps
template <int P, bool ALL, int DEST>
__device__ __forceinline__ void ortho_panel(const OrthoPanels& p, const OrthoOut& out,
                                            const PanelGroup& g, int matrix, int panel, lchar* lds) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int s = g.s, l = g.l;
  const int64_t at = (int64_t)matrix * panel_bytes(g);
  const char* rows = p.base + g.rows + at;
  const char* columns = p.base + g.columns + at;
  lchar* x = lds;
  lchar* y = x + P * PANEL * l * 2;
  lchar* a = y + P * PANEL * l * 2;
  const int dm = lane & 15, dn = 4 * (lane >> 4);

  const int j0 = wave * 16;
  PanelRows<P, P> r;
  PanelRows<P, 2> c;
  if (ALL && j0 < s) r.begin(rows, j0, l, lane);
  if (ALL && j0 < l) c.begin(columns, j0, s, lane);
  const char* mine = rows + (int64_t)panel * P * PANEL * l * 2;
  for (int i = threadIdx.x; i < P * PANEL * l / 8; i += PANEL_THREADS)
    ((lv4u*)x)[i] = (v4u_t)((const gv4u_a16*)mine)[i];
  // the panel t times X^T
  auto by_rows = [&](const lchar* t, float scale) {
    for (int j = j0; j < s; j += PANEL_WAVES * 16) {
      v4f u;
      if constexpr (ALL) u = r.product(t, lane);
      else u = panel_product<P, P>(rows, j, l, t, lane);
      panel_put<2>(a, dm, j + dn, u * scale);
    }
  };
  // the panel a times X
  auto by_columns = [&](int j) {
    if constexpr (ALL) return c.product(a, lane);
    else return panel_product<P, 2>(columns, j, s, a, lane);
  };
  __syncthreads();
  by_rows(x, p.gram);
  __syncthreads();
  v4f held[PANEL_BLOCKS];
#pragma unroll
  for (int h = 0; h < PANEL_BLOCKS; ++h) {
    const int j = j0 + h * PANEL_WAVES * 16;
    if (j >= l) break;
    held[h] = by_columns(j);
    panel_put<P>(y, dm, j + dn, held[h] * p.second);
  }
  __syncthreads();
  by_rows(y, p.third);
  __syncthreads();
  const int e = g.first + matrix, m = panel * PANEL + dm;
  char* next_rows = p.base + g.next_rows + at + (int64_t)panel * P * PANEL * l * 2;
  char* next_columns = p.base + g.next_columns + at;
#pragma unroll
  for (int h = 0; h < PANEL_BLOCKS; ++h) {
    const int j = j0 + h * PANEL_WAVES * 16, n = j + dn;
    if (j >= l) break;
    const v4f z = by_columns(j);
    v4f v = halves_to_v4f(SCAO_F16, small_pair(x + panel_at<P>(dm, n), 0));
    if constexpr (P == 2)
      v += halves_to_v4f(SCAO_F16, small_pair(x + panel_at<P>(dm, n) + 1024, 0));
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = fmaf(p.c, z[q], fmaf(p.b, held[h][q], p.a * v[q]));
    if (DEST == ORTHO_NEXT) {
      v2u w[P];
      ortho_words<P>(v, w);
      char* turned = next_columns + (int64_t)(j / 16) * P * PANEL * s * 2;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        *(gv2u_a8*)(next_rows + panel_at<P>(dm, n) + i * 1024) = w[i];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *(gu16*)(turned + panel_at<P>(dn + q, m) + i * 1024) =
              (uint16_t)(w[i][q / 2] >> (16 * (q & 1)));
      }
    } else if (m < g.source_s) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (n + q >= g.source_l) continue;
        const int64_t to = (int64_t)(g.wide ? m : n + q) * out.ld[e] + (g.wide ? n + q : m);
        float r = v[q];
        if (DEST == ORTHO_PARAMETER)
          r = fmaf(-out.rate[e], r, out.decay[e] * ld1(out.p[e], out.dt[e], to));
        st1(out.p[e], out.dt[e], to, r);
      }
    }
  }
}

template <bool ALL, int DEST>
__global__ __launch_bounds__(PANEL_THREADS) void k_ortho_panels(const OrthoPanels p,
                                                                const OrthoOut out) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  int in;
  const PanelGroup& g = panel_group(p.g, p.groups, in);
  const int matrix = in / g.per, panel = in % g.per;
  if (ALL || g.words == 1) ortho_panel<1, ALL, DEST>(p, out, g, matrix, panel, (lchar*)smem);
  else ortho_panel<2, false, DEST>(p, out, g, matrix, panel, (lchar*)smem);
}

// ------------------------------------------------------------ the first X ---
struct PanelSources {
  const void* src[ORTHO_MATRICES];
  const float* buf[ORTHO_MATRICES];   // the momentum behind its step, or null
  int ld[ORTHO_MATRICES];
  uint8_t dt[ORTHO_MATRICES];
  PanelGroup g[ORTHO_GROUPS];
  char* base;
  const double* norms;
  double eps, scale;
  float momentum, rest;
  int groups, nesterov;
};
static_assert(sizeof(PanelSources) <= 4096, "kernel arguments are limited to 4 KiB");

// 8 elements a thread in either order; what no source holds is zero
template <int P>
__device__ __forceinline__ void panel_first(const PanelSources& p, const PanelGroup& g, int matrix,
                                            int panel, double scale) {
  const int e = g.first + matrix, dt = p.dt[e], cols = g.wide ? g.source_l : g.source_s;
  const void* src = p.src[e];
  const float* buf = p.buf[e];
  const int64_t ld = p.ld[e], at = (int64_t)matrix * panel_bytes(g);
  auto value = [&](int m, int n) -> float {   // of row m of s, column n of l
    if (m >= g.source_s || n >= g.source_l) return 0.f;
    const int r = g.wide ? m : n, c = g.wide ? n : m;
    float u = ld1(src, dt, r * ld + c);
    if (buf) {
      const float now = gld1(buf + (int64_t)r * cols + c);
      u = p.nesterov ? fmaf(p.momentum, now, p.rest * u) : now;
    }
    return (float)((double)u * scale);
  };
  // a panel's rows, and its share of the columns
  const int units = PANEL * g.l / 8;
  for (int i = threadIdx.x; i < 2 * units; i += PANEL_THREADS) {
    const bool turned = i >= units;
    const int u = (turned ? i - units : i) + panel * units, lane = u % 64, piece = u / 64;
    const int across = (turned ? g.s : g.l) / 32;
    const int row = piece / across * 16 + lane % 16, k = piece % across * 32 + lane / 16 * 8;
    v4f v[2];
#pragma unroll
    for (int t = 0; t < 8; ++t) v[t / 4][t % 4] = turned ? value(k + t, row) : value(row, k + t);
    v2u w[2][P];
    ortho_words<P>(v[0], w[0]);
    ortho_words<P>(v[1], w[1]);
    char* to = p.base + (turned ? g.columns : g.rows) + at + (int64_t)piece * P * 1024 + lane * 16;
#pragma unroll
    for (int q = 0; q < P; ++q)
      *(gv4u_a16*)(to + q * 1024) = v4u_t{w[0][q][0], w[0][q][1], w[1][q][0], w[1][q][1]};
  }
}
__global__ __launch_bounds__(PANEL_THREADS) void k_panel_first(const PanelSources p) {
  __shared__ double lds[PANEL_WAVES], total;
  int in;
  const PanelGroup& g = panel_group(p.g, p.groups, in);
  const int matrix = in / g.per, panel = in % g.per;
  double s[1] = {0.0};
  for (int i = threadIdx.x; i < g.parts; i += PANEL_THREADS)
    s[0] += p.norms[(g.first + matrix) * ORTHO_PARTS + i];
  block_sum_n<1, PANEL_THREADS>(s, lds);
  if (threadIdx.x == 0) total = s[0];
  __syncthreads();
  const double norm = sqrt(total);
  const double scale = norm <= 1.7976931348623157e308 ? p.scale / (norm + p.eps) : norm - norm;
  if (g.words == 2) panel_first<2>(p, g, matrix, panel, scale);
  else panel_first<1>(p, g, matrix, panel, scale);
}

}  // namespace scao
