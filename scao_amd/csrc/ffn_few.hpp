// The gated feed-forward block's forward products for few tokens (serving):
// bound by reading the weights once.
//
// A workgroup owns 16 output columns (with GATED those of both projections) for
// all tokens; its NW waves share k, and their sums meet in LDS in a fixed
// order.  The weights go from global memory straight into the matrix cores'
// operand registers, 16 bytes (fp32: 32) a lane and step of 32 k: each byte is
// used once, so staging them would only add a trip.  All steps of a wave's run
// are independent loads, U of them in flight at a time.  Rows may start at any
// element and have any stride; the end of k is taken element by element.  fp32
// products are six products of bf16 parts, split in registers.
//
// HALVES (up to 8 tokens): the 16 rows and 16 columns of a product are 8 output
// columns and 8 tokens twice, for two different stretches of k; the quarters of
// the result where both belong together are added.  Twice as many workgroups
// with half the k each, for projections with few columns (one token, 8192 to 2048
// in bf16: 128 workgroups of 16 columns 12.0 us, 256 of 8 columns 8.3; 14336 to
// 4096 has enough, and loses 3 us of 71 in halves).
//
// Measured (bf16, weights not in the caches): one token, 4096 x 14336: 72 us,
// 4.9 TB/s of the 5.7 that a copy reaches; 2048 x 8192: 23 us of which 17.8 are
// the bytes.  From about 8 tokens on the tokens' operands cost as much address
// processing as the weights (16 rows of 64 bytes a load), and tiles win.
#pragma once

#include "ffn_kernels.hpp"

namespace scao {

struct FfnFew {
  const void* x;            // tokens x K
  const void* w;            // columns x K
  const void* w2;           // the up projection's with GATED
  int64_t ldx, ldw, ldw2;
  int tokens, cols, K;
};

typedef __attribute__((address_space(1))) v4u_t gv4u_any __attribute__((aligned(2)));

// eight consecutive elements as an operand
template <int TYPE>
struct Few8 {
  v4u_t q;
  static constexpr int SIZE = 2;
  __device__ void zero() { q = v4u_t{0, 0, 0, 0}; }
  __device__ void load(const char* p) { q = *(const gv4u_any*)p; }
  __device__ void load_some(const char* p, int n) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t lo = 2 * t < n ? ((const gu16*)p)[2 * t] : 0;
      const uint32_t hi = 2 * t + 1 < n ? ((const gu16*)p)[2 * t + 1] : 0;
      q[t] = lo | hi << 16;
    }
  }
  static __device__ v4f product(const Few8& w, const Few8& x, v4f c) {
    if (TYPE == SCAO_F16)
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, w.q),
                                                    __builtin_bit_cast(v8h, x.q), c, 0, 0, 0);
    return mfma16bf(__builtin_bit_cast(v8bf, w.q), __builtin_bit_cast(v8bf, x.q), c);
  }
};
template <>
struct Few8<SCAO_F32> {
  v4f a, b;
  static constexpr int SIZE = 4;
  __device__ void zero() { a = b = v4f{0.f, 0.f, 0.f, 0.f}; }
  __device__ void load(const char* p) {
    a = gld4((const float*)p);
    b = gld4((const float*)p + 4);
  }
  __device__ void load_some(const char* p, int n) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      a[t] = t < n ? gld1((const float*)p + t) : 0.f;
      b[t] = 4 + t < n ? gld1((const float*)p + 4 + t) : 0.f;
    }
  }
  __device__ bf3 split() const {
    const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return split_bf3(v);
  }
};

// U: steps in flight
template <int TYPE, int MT, int NW, int U, bool GATED, bool HALVES>
__global__ __launch_bounds__(NW * 64) void k_ffn_few(const FfnFew o, const FfnEpilogue e) {
  constexpr int H = GATED ? 2 : 1, P = HALVES ? 2 : 1, COLS_ = 16 / P;
  static_assert(!HALVES || MT == 1, "halves: one product of 16 x 16");
  __shared__ v4f sums[NW][H * MT][64];
  using V = Few8<TYPE>;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int q = lane & 15, g = lane >> 4;
  const int c0 = blockIdx.x * COLS_;
  const int row = HALVES ? q & 7 : q, half = HALVES ? q >> 3 : 0;

  // this lane's stretch of k steps, of the same length for all
  const int steps = (o.K + 31) / 32, per = (steps + NW * P - 1) / (NW * P);
  const int first = (wave * P + half) * per;
  // steps that are whole for every lane of the wave
  const int whole = min(per, o.K / 32 - (wave * P + P - 1) * per);

  // row starts; rows outside of the operands repeat the last one, their results
  // are never written
  const char *pw[H], *px[MT];
  const int64_t k0 = (int64_t)first * 32 + 8 * g;
  const int64_t r = min(c0 + row, o.cols - 1);
  pw[0] = (const char*)o.w + (r * o.ldw + k0) * V::SIZE;
  if (GATED) pw[H - 1] = (const char*)o.w2 + (r * o.ldw2 + k0) * V::SIZE;
#pragma unroll
  for (int m = 0; m < MT; ++m)
    px[m] = (const char*)o.x + ((int64_t)min(m * 16 + row, o.tokens - 1) * o.ldx + k0) * V::SIZE;

  v4f acc[H][MT];
#pragma unroll
  for (int i = 0; i < H; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[i][m] = v4f{0.f, 0.f, 0.f, 0.f};

  auto products = [&](const V (&w)[H], const V (&x)[MT]) {
    if constexpr (TYPE == SCAO_F32) {
      bf3 xs[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) xs[m] = x[m].split();
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const bf3 ws = w[i].split();
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[i][m] = mfma_x6(ws, xs[m], acc[i][m]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < H; ++i)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[i][m] = V::product(w[i], x[m], acc[i][m]);
    }
  };

  int s = 0;
  for (; s + U <= whole; s += U) {   // all lanes' steps are whole
    V w[U][H], x[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < H; ++i) w[u][i].load(pw[i] + (int64_t)(s + u) * 32 * V::SIZE);
#pragma unroll
      for (int m = 0; m < MT; ++m) x[u][m].load(px[m] + (int64_t)(s + u) * 32 * V::SIZE);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) products(w[u], x[u]);
  }
  // what is left of the stretch, and the end of k
  for (; s < per; s += U) {
    V w[U][H], x[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int left = s + u < per ? o.K - (first + s + u) * 32 - 8 * g : 0;
      const int64_t at = (int64_t)(s + u) * 32 * V::SIZE;
#pragma unroll
      for (int i = 0; i < H; ++i) w[u][i].zero();
#pragma unroll
      for (int m = 0; m < MT; ++m) x[u][m].zero();
      if (left >= 8) {
#pragma unroll
        for (int i = 0; i < H; ++i) w[u][i].load(pw[i] + at);
#pragma unroll
        for (int m = 0; m < MT; ++m) x[u][m].load(px[m] + at);
      } else if (left > 0) {
#pragma unroll
        for (int i = 0; i < H; ++i) w[u][i].load_some(pw[i] + at, left);
#pragma unroll
        for (int m = 0; m < MT; ++m) x[u][m].load_some(px[m] + at, left);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) products(w[u], x[u]);
  }

#pragma unroll
  for (int i = 0; i < H; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m) sums[wave][i * MT + m][lane] = acc[i][m];
  __syncthreads();
  for (int f = wave; f < MT; f += NW) {
    v4f a = {0.f, 0.f, 0.f, 0.f}, b = a;
    // HALVES: columns 4g .. 4g+3 of tokens 0 .. 7 (lanes with q < 8, g < 2) from
    // the first stretch, and 40 lanes further from the second
    if (HALVES && (q >= 8 || g >= 2)) return;
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int p = 0; p < P; ++p) {
        a += sums[w][f][lane + 40 * p];
        if (GATED) b += sums[w][MT + f][lane + 40 * p];
      }
    const int m = f * 16 + q, n = c0 + 4 * g;
    if constexpr (GATED) {
      v4f h;
      for_activation(e.act, [&](auto act) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          float v, d;
          activation<decltype(act)::value, TYPE == SCAO_F32>(a[t], v, d);
          h[t] = v * b[t];
        }
      });
      epi_store<TYPE>(e, m, n, h);
    } else {
      epi_store<TYPE>(e, m, n, a);
    }
  }
}

// most tokens that these kernels take
constexpr int FFN_FEW_TOKENS = 64;

template <int TYPE>
void launch_few(const FfnFew& o, const FfnEpilogue& e, bool gated, hipStream_t st) {
#define FFN_FEW(MT, NW, U, G, HALVES)                                  \
  k_ffn_few<TYPE, MT, NW, U, G, HALVES>                                 \
      <<<(o.cols + (HALVES ? 7 : 15)) / (HALVES ? 8 : 16), NW * 64, 0, st>>>(o, e)
  // halves where 16 columns a workgroup would not give every CU one
  const bool halves = o.tokens <= 8 && o.cols < 16 * 256;
  constexpr int U = TYPE == SCAO_F32 ? 4 : 8;
  if (gated) {
    if (halves) FFN_FEW(1, 8, U, true, true);
    else if (o.tokens <= 16) FFN_FEW(1, 8, U, true, false);
    else if (o.tokens <= 32) FFN_FEW(2, 8, TYPE == SCAO_F32 ? 2 : 4, true, false);
    else FFN_FEW(4, 8, 2, true, false);
  } else {
    if (halves) FFN_FEW(1, 16, U, false, true);
    else if (o.tokens <= 16) FFN_FEW(1, 16, U, false, false);
    else if (o.tokens <= 32) FFN_FEW(2, 16, TYPE == SCAO_F32 ? 2 : 4, false, false);
    else FFN_FEW(4, 8, TYPE == SCAO_F32 ? 2 : 4, false, false);
  }
#undef FFN_FEW
}

}  // namespace scao
