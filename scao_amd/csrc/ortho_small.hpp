// Small matrices, orthogonalised by one workgroup each in one launch: X and A stay in
// LDS as two fp16 words an element from the first norm to the result.
//
// A tile's beginning and end and a launch's own time are nearly all of a small
// product: a call of 2 + 3 launches a step takes 8 us a launch whatever it multiplies.
// Here a step is three passes over LDS.  Five steps of 32 x 32 take 16 us, of 64 x 64
// 21, 96 x 96 37, 128 x 128 65 (by tiles 135 and more, by panels 34, 37, 43 and 49);
// 32 matrices as long as one.
// Bound by LDS reads (a fragment of either operand, 4 KB, for three 16 x 16 x 32
// products) and their latency: eight waves instead of sixteen take half as long again.
//
//   X  s x l, rows of l (tall matrices are turned as they are read), zeros up to whole
//      steps of 32 either way.  A's products read its rows, an update's its columns,
//      by LDS reads that transpose; a wave's update needs no columns but its own, so
//      they are replaced in place.
//   A  s x s, replaced by B once every wave holds its share of A A in registers.
//
// Rows are an odd number of 16-byte pieces long, so that 16 rows' pieces lie in
// different banks.
#pragma once

#include "ortho_norm.hpp"

namespace scao {

constexpr int SMALL_SIDE = 128;
constexpr int SMALL_STEPS = 16;
constexpr int SMALL_THREADS = 1024, SMALL_WAVES = SMALL_THREADS / 64;
constexpr int SMALL_LDS = 156 * 1024;
struct OrthoSmall {
  const void* src[ORTHO_MATRICES];
  float* buf[ORTHO_MATRICES];
  void* dst[ORTHO_MATRICES];
  int rows[ORTHO_MATRICES], cols[ORTHO_MATRICES], ld_src[ORTHO_MATRICES], ld_dst[ORTHO_MATRICES];
  float rate[ORTHO_MATRICES], decay[ORTHO_MATRICES];
  uint8_t src_dt[ORTHO_MATRICES], dst_dt[ORTHO_MATRICES];
  float gram[SMALL_STEPS], square[SMALL_STEPS], keep[SMALL_STEPS], diagonal[SMALL_STEPS],
      update[SMALL_STEPS];
  double eps, scale;
  float momentum, rest;
  int steps, nesterov;
};
static_assert(sizeof(OrthoSmall) <= 4096, "kernel arguments are limited to 4 KiB");

// elements of a row of n in LDS
__host__ __device__ inline int small_row(int n) { return ((n + 31) / 32 * 4 | 1) * 8; }
__host__ __device__ inline int small_lds(int s, int l) {
  const int sp = (s + 31) / 32 * 32;
  return 4 * sp * (small_row(l) + small_row(s));
}

// 16 rows from r0, k = k0 .. k0 + 31, of rows of ld
__device__ __forceinline__ v8s small_rows(const lchar* t, int ld, int r0, int k0, int lane) {
  return *(const lv8s*)(t + ((r0 + (lane & 15)) * ld + k0 + 8 * (lane >> 4)) * 2);
}
// the same of columns: 16 columns from r0
__device__ __forceinline__ v8s small_columns(const lchar* t, int ld, int r0, int k0, int lane) {
  const int q = lane & 15, k = k0 + 8 * (lane >> 4) + (q >> 2);
  const lchar* p = t + (k * ld + r0 + (q & 3) * 4) * 2;
  const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lv4s*)p);
  const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lv4s*)(p + 4 * ld * 2));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
// the three products of words in sums of their own, so that none waits for another
struct SmallSum {
  v4f c[3] = {};
  __device__ __forceinline__ void add(const v8s (&p)[2], const v8s (&q)[2]) {
    c[0] = mma<true>(p[1], q[0], c[0]);
    c[1] = mma<true>(p[0], q[1], c[1]);
    c[2] = mma<true>(p[0], q[0], c[2]);
  }
  // rows from i times rows from j of one matrix, STEPS steps of k from k on, all of
  // their reads ahead of the products
  template <int STEPS>
  __device__ __forceinline__ void rows(const lchar* t, int plane, int ld, int i, int j, int k,
                                       int lane) {
    v8s u[STEPS][2], v[STEPS][2];
#pragma unroll
    for (int h = 0; h < STEPS; ++h)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        u[h][w] = small_rows(t + w * plane * 2, ld, i, k + 32 * h, lane);
        v[h][w] = small_rows(t + w * plane * 2, ld, j, k + 32 * h, lane);
      }
#pragma unroll
    for (int h = 0; h < STEPS; ++h) add(u[h], v[h]);
  }
  __device__ __forceinline__ v4f value() const { return (c[0] + c[1]) + c[2]; }
};
typedef __attribute__((address_space(3))) v2u lv2u;
typedef __attribute__((address_space(3))) uint16_t lu16;
__device__ __forceinline__ v2u small_pair(const lchar* t, int at) { return *(const lv2u*)(t + at * 2); }

// fragment f of those on and below the diagonal
__device__ __forceinline__ void small_fragment(int f, int& i, int& j) {
  i = 0;
  while ((i + 1) * (i + 2) / 2 <= f) ++i;
  j = f - i * (i + 1) / 2;
}
// A[m][n .. n + 3] and its mirror image
__device__ __forceinline__ void small_put(lchar* a, int plane, int ld, int m, int n, bool mirror,
                                          v4f c) {
  v2u w[2];
  ortho_words<2>(c, w);
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    *(lv2u*)(a + (p * plane + m * ld + n) * 2) = w[p];
    if (mirror)
#pragma unroll
      for (int t = 0; t < 4; ++t)
        *(lu16*)(a + (p * plane + (n + t) * ld + m) * 2) = (uint16_t)(w[p][t / 2] >> (16 * (t & 1)));
  }
}

// What one workgroup works on.
struct SmallMatrix {
  lchar *x, *a;              // in LDS
  int s, l, ldx, lda, px, pa;   // px, pa: elements of a plane
  int rows, cols, wave, lane;
  bool wide;
};

// X from the source of type DT: the update, eight elements a thread under way; its
// squares' sum, and its fp32 values in the places of X's words (half in either) until
// the norm is known.
template <int DT>
__device__ __forceinline__ void small_begin(const OrthoSmall& p, const SmallMatrix& t, int e,
                                            double* sums) {
  const void* src = p.src[e];
  float* buf = p.buf[e];
  const int ld_src = p.ld_src[e], all = t.rows * t.cols;
  // (exact: fewer than 2^21 elements, and i + 1/2 is at least 1/2 from a multiple)
  const float per_row = 1.f / t.cols;
  auto row_of = [&](int i) { return (int)((i + 0.5f) * per_row); };
  auto place = [&](int i, int r) {
    const int c = i - r * t.cols;
    return t.wide ? r * t.ldx + c : c * t.ldx + r;
  };
  double square[1] = {0.0};
  constexpr int AHEAD = 8;
  for (int i0 = threadIdx.x; i0 < all; i0 += AHEAD * SMALL_THREADS) {
    float g[AHEAD], m[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {   // (past the end the last element again)
      const int i = min(i0 + k * SMALL_THREADS, all - 1), r = row_of(i);
      g[k] = ld1(src, DT, (int64_t)r * ld_src + i - r * t.cols);
    }
    if (buf)
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) m[k] = gld1(buf + min(i0 + k * SMALL_THREADS, all - 1));
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = i0 + k * SMALL_THREADS;
      if (i >= all) break;
      float u = g[k];
      if (buf) {
        const float part = p.rest * u;
        m[k] = fmaf(p.momentum, m[k], part);
        gst1(buf + i, m[k]);
        u = p.nesterov ? fmaf(p.momentum, m[k], part) : m[k];
      }
      square[0] = fma((double)u, (double)u, square[0]);
      const int at = place(i, row_of(i));
      *(lu16*)(t.x + at * 2) = (uint16_t)(__float_as_uint(u) >> 16);
      *(lu16*)(t.x + (t.px + at) * 2) = (uint16_t)__float_as_uint(u);
    }
  }
  block_sum_n<1, SMALL_THREADS>(square, sums);
  if (threadIdx.x == 0) sums[0] = square[0];
  __syncthreads();
  const double norm = sqrt(sums[0]);
  const double scale = norm <= 1.7976931348623157e308 ? p.scale / (norm + p.eps) : norm - norm;
  for (int i = threadIdx.x; i < all; i += SMALL_THREADS) {
    const int at = place(i, row_of(i));
    lu16 *high = (lu16*)(t.x + at * 2), *low = (lu16*)(t.x + (t.px + at) * 2);
    const float v = (float)((double)__uint_as_float((uint32_t)*high << 16 | *low) * scale);
    const uint16_t hi = f_to_f16(v);
    *high = hi;
    *low = f_to_f16(v - f16_to_f(hi));
  }
  __syncthreads();
}

// All steps of a matrix whose smaller side is up to 32 KS.
template <int KS, int DEST>
__device__ __forceinline__ void small_steps(const OrthoSmall& p, const SmallMatrix& t, int e) {
  constexpr int SIDE = 2 * KS, LOWER = SIDE * (SIDE + 1) / 2;
  constexpr int HELD = (LOWER + SMALL_WAVES - 1) / SMALL_WAVES;   // fragments of A a wave has
  lchar *x = t.x, *a = t.a;
  const int ldx = t.ldx, lda = t.lda, px = t.px, pa = t.pa, lane = t.lane, wave = t.wave;
  const int dm = lane & 15, dn = 4 * (lane >> 4);
  int fi[HELD], fj[HELD];
#pragma unroll
  for (int h = 0; h < HELD; ++h) small_fragment(min(wave + h * SMALL_WAVES, LOWER - 1), fi[h], fj[h]);
  auto mine = [&](int h) { return wave + h * SMALL_WAVES < LOWER; };

  for (int step = 0; step < p.steps; ++step) {
    // A = X X^T
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      if (!mine(h)) continue;
      SmallSum sum;
      int k = 0;
      for (; k + 96 < t.l; k += 128) sum.rows<4>(x, px, ldx, fj[h] * 16, fi[h] * 16, k, lane);
      for (; k < t.l; k += 32) sum.rows<1>(x, px, ldx, fj[h] * 16, fi[h] * 16, k, lane);
      small_put(a, pa, lda, fi[h] * 16 + dm, fj[h] * 16 + dn, fi[h] != fj[h],
                sum.value() * p.gram[step]);
    }
    __syncthreads();
    // B = diagonal + keep A + A A
    v4f held[HELD];
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      if (!mine(h)) continue;
      const int m = fi[h] * 16 + dm, n = fj[h] * 16 + dn;
      SmallSum sum;
      const v2u add[2] = {small_pair(a, m * lda + n), small_pair(a, pa + m * lda + n)};
      sum.rows<KS>(a, pa, lda, fj[h] * 16, fi[h] * 16, 0, lane);
      v4f c = sum.value() * p.square[step];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const v4f y = halves_to_v4f(SCAO_F16, add[w]);
#pragma unroll
        for (int q = 0; q < 4; ++q) c[q] = fmaf(p.keep[step], y[q], c[q]);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (n + q == m && m < t.s) c[q] += p.diagonal[step];
      held[h] = c;
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < HELD; ++h)
      if (mine(h))
        small_put(a, pa, lda, fi[h] * 16 + dm, fj[h] * 16 + dn, fi[h] != fj[h], held[h]);
    __syncthreads();
    // X <- B X, 16 columns a wave; few columns: shared by several waves, which take
    // rows in turns once all of them have read theirs
    const bool last = step + 1 == p.steps;
    const int blocks = (t.l + 15) / 16, sharing = blocks < SMALL_WAVES ? SMALL_WAVES / blocks : 1;
    for (int b = wave / sharing; b < blocks || b == wave / sharing; b += SMALL_WAVES / sharing) {
      const int c0 = min(b, blocks - 1) * 16;
      v8s u[KS][2];
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        u[k][0] = small_columns(x, ldx, c0, k * 32, lane);
        u[k][1] = small_columns(x + px * 2, ldx, c0, k * 32, lane);
      }
      if (sharing > 1) __syncthreads();
      if (b >= blocks) break;
      for (int i = wave % sharing; i < SIDE; i += sharing) {
        v8s v[KS][2];
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          v[k][0] = small_rows(a, lda, i * 16, k * 32, lane);
          v[k][1] = small_rows(a + pa * 2, lda, i * 16, k * 32, lane);
        }
        SmallSum sum;
#pragma unroll
        for (int k = 0; k < KS; ++k) sum.add(u[k], v[k]);
        const v4f c = sum.value() * p.update[step];
        const int m = i * 16 + dm, n = c0 + dn;
        if (!last) {
          v2u w[2];
          ortho_words<2>(c, w);
          *(lv2u*)(x + (m * ldx + n) * 2) = w[0];
          *(lv2u*)(x + (px + m * ldx + n) * 2) = w[1];
        } else if (m < t.s) {
          const int out = p.dst_dt[e];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (n + q >= t.l) continue;
            const int64_t at = (int64_t)(t.wide ? m : n + q) * p.ld_dst[e] + (t.wide ? n + q : m);
            float y = c[q];
            if (DEST == ORTHO_PARAMETER)
              y = fmaf(-p.rate[e], y, p.decay[e] * ld1(p.dst[e], out, at));
            st1(p.dst[e], out, at, y);
          }
        }
      }
    }
    __syncthreads();
  }
}

template <int DEST>
__global__ __launch_bounds__(SMALL_THREADS) void k_ortho_small(const OrthoSmall p) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  __shared__ double sums[SMALL_WAVES];
  const int e = blockIdx.x;
  SmallMatrix t;
  t.rows = p.rows[e];
  t.cols = p.cols[e];
  t.wide = t.rows <= t.cols;
  t.s = t.wide ? t.rows : t.cols;
  t.l = t.wide ? t.cols : t.rows;
  const int ks = (t.s + 31) / 32;
  t.ldx = small_row(t.l);
  t.lda = small_row(t.s);
  t.px = ks * 32 * t.ldx;
  t.pa = ks * 32 * t.lda;
  t.x = (lchar*)smem;
  t.a = t.x + 4 * t.px;
  t.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  t.lane = threadIdx.x & 63;

  typedef __attribute__((address_space(3))) v4u_t lv4u;
  for (int i = threadIdx.x; i < (t.px + t.pa) / 4; i += SMALL_THREADS)
    ((lv4u*)t.x)[i] = v4u_t{0, 0, 0, 0};
  __syncthreads();
  const int dt = p.src_dt[e];
  if (dt == SCAO_F32) small_begin<SCAO_F32>(p, t, e, sums);
  else if (dt == SCAO_BF16) small_begin<SCAO_BF16>(p, t, e, sums);
  else small_begin<SCAO_F16>(p, t, e, sums);
  if (ks == 1) small_steps<1, DEST>(p, t, e);
  else if (ks == 2) small_steps<2, DEST>(p, t, e);
  else if (ks == 3) small_steps<3, DEST>(p, t, e);
  else small_steps<4, DEST>(p, t, e);
}

}  // namespace scao
