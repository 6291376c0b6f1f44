// The gated feed-forward block's forward products for few tokens (serving):
// bound by reading the weights once.
//
// A workgroup owns NR x 16 output columns (with GATED those of both projections)
// for all tokens; its NW waves share k, and their sums meet in LDS in a fixed
// order.  The weights go from global memory straight into the matrix cores'
// operand registers, 16 bytes (fp32: 32) a lane and step of 32 k: each byte is
// used once, so staging them would only add a trip.  All steps of a wave's run
// are independent loads, U of them in flight at a time.  Rows may start at any
// element and have any stride; the end of k is taken element by element.  fp32
// products are six products of bf16 parts, split in registers.
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
template <int TYPE, int MT, int NR, int NW, int U, bool GATED>
__global__ __launch_bounds__(NW * 64) void k_ffn_few(const FfnFew o, const FfnEpilogue e) {
  constexpr int H = GATED ? 2 : 1, NF = MT * NR * H;
  __shared__ v4f sums[NW][NF][64];
  using V = Few8<TYPE>;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int q = lane & 15, g = lane >> 4;
  const int c0 = blockIdx.x * NR * 16;

  // row starts; rows outside of the operands repeat the last one, their results
  // are never written
  const char *pw[NR * H], *px[MT];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int64_t r = min(c0 + i * 16 + q, o.cols - 1);
    pw[i] = (const char*)o.w + (r * o.ldw + 8 * g) * V::SIZE;
    if (GATED) pw[NR * (H - 1) + i] = (const char*)o.w2 + (r * o.ldw2 + 8 * g) * V::SIZE;
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
    px[m] = (const char*)o.x + ((int64_t)min(m * 16 + q, o.tokens - 1) * o.ldx + 8 * g) * V::SIZE;

  v4f acc[NR * H][MT];
#pragma unroll
  for (int i = 0; i < NR * H; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[i][m] = v4f{0.f, 0.f, 0.f, 0.f};

  auto products = [&](const V (&w)[NR * H], const V (&x)[MT]) {
    if constexpr (TYPE == SCAO_F32) {
      bf3 xs[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) xs[m] = x[m].split();
#pragma unroll
      for (int i = 0; i < NR * H; ++i) {
        const bf3 ws = w[i].split();
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[i][m] = mfma_x6(ws, xs[m], acc[i][m]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NR * H; ++i)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[i][m] = V::product(w[i], x[m], acc[i][m]);
    }
  };

  const int steps = (o.K + 31) / 32, whole = o.K / 32;
  const int per = (steps + NW - 1) / NW;
  int s = wave * per;
  const int end = min(steps, s + per), full = min(whole, end);
  for (; s + U <= full; s += U) {
    V w[U][NR * H], x[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < NR * H; ++i) w[u][i].load(pw[i] + (int64_t)(s + u) * 32 * V::SIZE);
#pragma unroll
      for (int m = 0; m < MT; ++m) x[u][m].load(px[m] + (int64_t)(s + u) * 32 * V::SIZE);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) products(w[u], x[u]);
  }
  for (; s < end; ++s) {
    V w[NR * H], x[MT];
    const int left = o.K - s * 32 - 8 * g;
#pragma unroll
    for (int i = 0; i < NR * H; ++i) {
      const char* p = pw[i] + (int64_t)s * 32 * V::SIZE;
      if (s < full) w[i].load(p);
      else w[i].load_some(p, left);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const char* p = px[m] + (int64_t)s * 32 * V::SIZE;
      if (s < full) x[m].load(p);
      else x[m].load_some(p, left);
    }
    products(w, x);
  }

#pragma unroll
  for (int i = 0; i < NR * H; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m) sums[wave][i * MT + m][lane] = acc[i][m];
  __syncthreads();
  for (int f = wave; f < NR * MT; f += NW) {
    v4f a = sums[0][f][lane], b = sums[0][NR * MT * (H - 1) + f][lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) {
      a += sums[w][f][lane];
      if (GATED) b += sums[w][NR * MT + f][lane];
    }
    const int m = (f % MT) * 16 + q, n = c0 + (f / MT) * 16 + 4 * g;
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
#define FFN_FEW(MT, NR, NW, U, G) \
  k_ffn_few<TYPE, MT, NR, NW, U, G><<<(o.cols + NR * 16 - 1) / (NR * 16), NW * 64, 0, st>>>(o, e)
  if (gated) {
    if (o.tokens <= 16) FFN_FEW(1, 1, 8, 4, true);
    else if (o.tokens <= 32) FFN_FEW(2, 1, 8, 4, true);
    else FFN_FEW(4, 1, 8, 2, true);
  } else {
    if (o.tokens <= 16) FFN_FEW(1, 1, 16, 4, false);
    else if (o.tokens <= 32) FFN_FEW(2, 1, 16, 4, false);
    else FFN_FEW(4, 1, 8, 4, false);
  }
#undef FFN_FEW
}

}  // namespace scao
