// From updates to the first X: the sums of squares of every matrix (of the
// optimiser's update, with the momentum's own step), and X = G / (|G| + eps) in
// fp16 words.  Two passes, as no element can be scaled before the last is summed; both
// bound by HBM (134 M elements of eight 8192 x 2048 with bf16 gradients: 257 us with
// the momentum's step, 5.2 TB/s, and 237, 4.5 TB/s; without four vectors under way and
// with 256 workgroups a matrix instead of 1024, 58.7 M elements alone took 79 and 95 us
// and now take 34 and 51), and short beside the products.
#pragma once

#include "ortho_kernels.hpp"

namespace scao {

// ------------------------------------------------------------- norms -------
// The sources are walked in units of 256 vectors of 8 elements: a piece of one
// row, or several short rows; a workgroup takes `per` units of one matrix.
struct OrthoSource {
  int rows, cols, ldx;
  int first, words;          // entry of the tables; 1 or 2 words an element
  int vecs;                  // vectors of a row side by side in a unit (a power of two)
  int across, per, parts;    // units a row, units a workgroup, workgroups a matrix
  int block0;                // workgroups of the groups before
  int64_t x, x_step;
};
struct OrthoPrep {
  const void* src[ORTHO_MATRICES];
  float* buf[ORTHO_MATRICES];   // momentum, or null
  int ld[ORTHO_MATRICES];
  uint8_t dt[ORTHO_MATRICES];
  OrthoSource g[ORTHO_GROUPS];
  char* base;
  double* norms;             // ORTHO_PARTS a matrix
  double eps, scale;
  float momentum, rest;      // mu, 1 - mu
  int groups, nesterov;
};

struct OrthoVector {
  v4f x[2];
};
// Eight elements from column c of row r.
template <int DT>
__device__ __forceinline__ OrthoVector ortho_load(const void* p, int64_t ld, int r, int c, int cols) {
  OrthoVector v;
  const int left = cols - c;
  const int64_t at = (int64_t)r * ld + c;
  if (left >= 8 && DT != SCAO_F32) {
    const v4u_t w = *(const gv4u_a2*)((const uint16_t*)p + at);
    v.x[0] = halves_to_v4f(DT, v2u{w[0], w[1]});
    v.x[1] = halves_to_v4f(DT, v2u{w[2], w[3]});
    return v;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int n = left - 4 * h;
    v.x[h] = ld4(p, DT, at + 4 * h, n >= 4, n <= 0 ? 0 : (1 << n) - 1);
  }
  return v;
}
__device__ __forceinline__ OrthoVector ortho_load_momentum(const float* buf, int cols, int r, int c) {
  OrthoVector v;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int n = cols - c - 4 * h;
    v.x[h] = ldf4(buf, (int64_t)r * cols + c + 4 * h, n >= 4, n <= 0 ? 0 : (1 << n) - 1);
  }
  return v;
}
// g becomes the update of momentum and gradient; NORM: the momentum takes its step
template <bool NORM>
__device__ __forceinline__ void ortho_momentum(const OrthoPrep& p, float* buf, int r, int c, int cols,
                                               OrthoVector& g, OrthoVector& m) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const float s = p.rest * g.x[h][t];
      if (NORM) m.x[h][t] = fmaf(p.momentum, m.x[h][t], s);
      g.x[h][t] = p.nesterov ? fmaf(p.momentum, m.x[h][t], s) : m.x[h][t];
    }
    const int n = cols - c - 4 * h;
    if (NORM)
      stf4(buf, (int64_t)r * cols + c + 4 * h, m.x[h], n >= 4, n <= 0 ? 0 : (1 << n) - 1);
  }
}

// f(row, column, vector) for the vectors of this thread, four of them loaded at a time
template <int DT, bool NORM, class F>
__device__ __forceinline__ void ortho_walk(const OrthoPrep& p, const OrthoSource& g, int matrix,
                                           int part, int width, F&& f) {
  constexpr int AHEAD = 4;
  const int rows_a_unit = 256 / g.vecs;
  const int units = (g.rows + rows_a_unit - 1) / rows_a_unit * g.across;
  const int begin = part * g.per, end = min(units, begin + g.per);
  const int v = threadIdx.x & (g.vecs - 1), rr = threadIdx.x / g.vecs;
  const void* src = p.src[g.first + matrix];
  float* buf = p.buf[g.first + matrix];
  const int64_t ld = p.ld[g.first + matrix];
  for (int u = begin; u < end; u += AHEAD) {
    OrthoVector x[AHEAD], m[AHEAD];
    int r[AHEAD], c[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      r[i] = (u + i) / g.across * rows_a_unit + rr;
      c[i] = ((u + i) % g.across * g.vecs + v) * 8;
      if (u + i >= end || r[i] >= g.rows) c[i] = width;
      if (c[i] < width) {
        x[i] = ortho_load<DT>(src, ld, r[i], c[i], g.cols);
        if (buf) m[i] = ortho_load_momentum(buf, g.cols, r[i], c[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (c[i] < width) {
        if (buf) ortho_momentum<NORM>(p, buf, r[i], c[i], g.cols, x[i], m[i]);
        f(r[i], c[i], x[i]);
      }
  }
}
template <bool NORM, class F>
__device__ __forceinline__ void ortho_walk(const OrthoPrep& p, const OrthoSource& g, int matrix,
                                           int part, int width, F&& f) {
  const int dt = p.dt[g.first + matrix];
  if (dt == SCAO_F32) ortho_walk<SCAO_F32, NORM>(p, g, matrix, part, width, f);
  else if (dt == SCAO_BF16) ortho_walk<SCAO_BF16, NORM>(p, g, matrix, part, width, f);
  else ortho_walk<SCAO_F16, NORM>(p, g, matrix, part, width, f);
}
__device__ __forceinline__ const OrthoSource& ortho_source(const OrthoPrep& p, int& matrix,
                                                           int& part) {
  int k = 0;
  for (int i = 1; i < p.groups; ++i)
    if ((int)blockIdx.x >= p.g[i].block0) k = i;
  const int in = blockIdx.x - p.g[k].block0;
  matrix = in / p.g[k].parts;
  part = in % p.g[k].parts;
  return p.g[k];
}

// sums of squares in double: no square of a float overflows or vanishes there
__global__ __launch_bounds__(256) void k_ortho_norm(const OrthoPrep p) {
  __shared__ double lds[4];
  int matrix, part;
  const OrthoSource& g = ortho_source(p, matrix, part);
  double s[1] = {0.0};
  ortho_walk<true>(p, g, matrix, part, g.cols, [&](int, int, const OrthoVector& x) {
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const double d = (double)x.x[t / 4][t % 4];
      s[0] = fma(d, d, s[0]);
    }
  });
  block_sum(s, lds);
  if (threadIdx.x == 0) p.norms[(g.first + matrix) * ORTHO_PARTS + part] = s[0];
}

// X, with zeros up to its row stride's end; NaN throughout where the norm is none
template <int P>
__device__ __forceinline__ void ortho_scale(const OrthoPrep& p, const OrthoSource& g, int matrix,
                                            int part, double scale) {
  uint16_t* x = (uint16_t*)(p.base + g.x + matrix * g.x_step);
  ortho_walk<false>(p, g, matrix, part, g.ldx, [&](int r, int c, const OrthoVector& u) {
    v2u w[2][P];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      v4f y;
#pragma unroll
      for (int t = 0; t < 4; ++t)
        y[t] = c + 4 * h + t < g.cols ? (float)((double)u.x[h][t] * scale) : 0.f;
      ortho_words<P>(y, w[h]);
    }
#pragma unroll
    for (int i = 0; i < P; ++i)
      *(gv4u_a16*)(x + ((int64_t)r * P + i) * g.ldx + c) =
          v4u_t{w[0][i][0], w[0][i][1], w[1][i][0], w[1][i][1]};
  });
}
__global__ __launch_bounds__(256) void k_ortho_scale(const OrthoPrep p) {
  __shared__ double lds[4], total;
  int matrix, part;
  const OrthoSource& g = ortho_source(p, matrix, part);
  double s[1] = {0.0};
  for (int i = threadIdx.x; i < g.parts; i += 256)
    s[0] += p.norms[(g.first + matrix) * ORTHO_PARTS + i];
  block_sum(s, lds);
  if (threadIdx.x == 0) total = s[0];
  __syncthreads();
  const double norm = sqrt(total);
  const double scale = norm <= 1.7976931348623157e308 ? p.scale / (norm + p.eps) : norm - norm;
  if (g.words == 2) ortho_scale<2>(p, g, matrix, part, scale);
  else ortho_scale<1>(p, g, matrix, part, scale);
}

}  // namespace scao
