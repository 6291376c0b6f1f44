// The kernels of the gated feed-forward block: the tiled products with their
// epilogues, the join of a product that was split over k, and the packing of
// operands.  One translation unit instantiates them for each type.
//
//   a = x Wg^T, b = x Wu^T, h = f(a) * b, y = h Wd^T
//   dh = dy Wd, da = dh * b * f'(a), db = dh * f(a)
//   dx = da Wg + db Wu, dWg = da^T x, dWu = db^T x, dWd = dy^T h
//
// Roundings of the 16-bit types: h, da and db, which enter further products on
// the matrix cores, to the type itself, once each; nothing else before the
// outputs.  a and b, which only enter f' and elementwise products, are kept for
// the backward pass with 16 significant bits (a float without its lowest byte):
// rounded to 8 (bf16) they would add as much error to da and db as those' own
// rounding.  In fp32 nothing is rounded below it (GELU's polynomial aside, which
// is good to 1.5e-7 of erfc): h, da and db are kept as three bf16 parts that add
// up to them, and a product of two such sums is six products of parts (see
// mfma_x6) run as six segments of one bf16 product.
#pragma once

#include "ffn_gemm.hpp"

namespace scao {

enum { EPI_STORE = 0, EPI_GATED = 1, EPI_DACT = 2 };

struct FfnEpilogue {
  void* out;            // STORE: rows of C; GATED: h; DACT: da, and db next to it
  void* out2;           // STORE: rows from `second` on, or null
  int64_t ldo;
  int64_t plane;        // GATED, DACT in fp32: elements from one part to the next
  int rows, second;     // STORE: rows of either output, C's row where the second begins
  int cols;             // columns written
  int fi, fj;           // fragments of 16 rows and of 16 columns of a and b kept
  void* ab;             // a and b by fragments, or null (GATED: nothing is kept)
  int act;
  float* partial;       // split products: the parts, by fragments
};

// ------------------------------------------------------- activations -------
// 1 / (1 + exp(-z)) from the hardware's exp2 and reciprocal (an ulp each).  The
// product z log2(e) is kept as a sum of two floats where the result is fp32:
// its rounding alone would be |z| 6e-8 of the result.
template <bool F32>
__device__ __forceinline__ float logistic(float z) {
  constexpr float L2E = 1.44269504f, L2E_LO = 1.92596303e-8f;
  float e;
  const float t = -z * L2E;
  if (F32) {
    const float lo = fmaf(-z, L2E, -t) - z * L2E_LO;
    // the correction only where it is a number (t finite) and matters
    const float p = __builtin_amdgcn_exp2f(t);
    e = fabsf(t) < 126.f ? fmaf(p, lo * 0.69314718f, p) : p;
  } else {
    e = __builtin_amdgcn_exp2f(t);
  }
  return __builtin_amdgcn_rcpf(1.f + e);
}

// f(a) and f'(a)
template <int ACT, bool F32>
__device__ __forceinline__ void activation(float a, float& f, float& g) {
  if (ACT == SCAO_ACT_SILU) {
    const float s = logistic<F32>(a);
    f = a * s;
    g = s * fmaf(a, 1.f - s, 1.f);
  } else if (ACT == SCAO_ACT_SIGMOID) {
    const float s = logistic<F32>(a);
    f = s;
    g = s * (1.f - s);
  } else if (ACT == SCAO_ACT_RELU) {
    f = a > 0.f || a != a ? a : 0.f;   // a NaN stays one, minus infinity does not become one
    g = a > 0.f ? 1.f : 0.f;
  } else if (ACT == SCAO_ACT_GELU) {
    // erfc(z) = t (a1 + t (a2 + ... )) exp(-z^2), t = 1 / (1 + 0.3275911 z), z >= 0,
    // to 1.5e-7 (Abramowitz and Stegun, Handbook of Mathematical Functions,
    // 7.1.26); exp(-z^2) = exp(-a^2/2) is the derivative's too
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678f, fabsf(a), 1.f));
    const float ex = __builtin_amdgcn_exp2f(-0.72134752f * (a * a));
    float p = fmaf(t, 1.061405429f, -1.453152027f);
    p = fmaf(t, p, 1.421413741f);
    p = fmaf(t, p, -0.284496736f);
    p = fmaf(t, p, 0.254829592f);
    const float tail = 0.5f * p * t * ex;
    const float c = a < 0.f ? tail : 1.f - tail;
    f = a * c;
    g = fmaf(a * 0.39894228f, ex, c);
  } else {   // a/2 (1 + tanh u) = a logistic(2u), u = sqrt(2/pi) (a + 0.044715 a^3)
    const float a2 = a * a;
    const float s = logistic<F32>(1.59576912f * fmaf(0.044715f * a2, a, a));
    f = a * s;
    g = fmaf(a * s * (1.f - s), 1.59576912f * fmaf(0.134145f, a2, 1.f), s);
  }
}

// --------------------------------------------------------- stores ----------
// TYPE: enum scao_dtype of the block.  Four values of one row as 16-bit words of
// each plane of an operand: the value, or (fp32) its three bf16 parts.
template <int TYPE>
constexpr int PLANES = TYPE == SCAO_F32 ? 3 : 1;
template <int TYPE>
__device__ __forceinline__ void operand_words(v4f x, v2u (&w)[PLANES<TYPE>]) {
  if constexpr (TYPE == SCAO_F32) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t h, m, l;
      split3_pk(x[2 * t], x[2 * t + 1], h, m, l);
      w[0][t] = h;
      w[1][t] = m;
      w[2][t] = l;
    }
  } else if (TYPE == SCAO_BF16) {
    w[0] = v2u{pk_bf16(x[0], x[1]), pk_bf16(x[2], x[3])};
  } else {
    w[0] = v4f_to_halves(SCAO_F16, x);
  }
}
template <int TYPE>
__device__ __forceinline__ void put_operand(void* base, int64_t at, int64_t plane, v4f x) {
  v2u w[PLANES<TYPE>];
  operand_words<TYPE>(x, w);
#pragma unroll
  for (int i = 0; i < PLANES<TYPE>; ++i) *(gv2u*)((uint16_t*)base + at + i * plane) = w[i];
}

// Two fragments next to each other: lane group g (16 lanes) holds columns 4g ..
// 4g+3 of either.  The odd groups of the first change places with the even ones
// of the second, after which a lane holds eight columns in order, those from
// pair_column(lane) on: one 16-byte store, 64 bytes of a row side by side.
__device__ __forceinline__ int pair_column(int lane) {
  return (lane >> 4 & 1) * 16 + (lane >> 5) * 8;
}
__device__ __forceinline__ v4u_t join_pair(v2u p, v2u q) {
  const auto a = __builtin_amdgcn_permlane16_swap(p[0], q[0], false, false);
  const auto b = __builtin_amdgcn_permlane16_swap(p[1], q[1], false, false);
  return v4u_t{a[0], b[0], a[1], b[1]};
}
typedef __attribute__((address_space(1))) v4u_t gv4u_a16;
typedef v4u_t v4u_a2 __attribute__((aligned(2)));
typedef __attribute__((address_space(1))) v4u_a2 gv4u_a2;
// at: the element of this lane's first column
template <int TYPE>
__device__ __forceinline__ void put_operand_pair(void* base, int64_t at, int64_t plane, bool in,
                                                 v4f x, v4f y) {
  v2u p[PLANES<TYPE>], q[PLANES<TYPE>];
  operand_words<TYPE>(x, p);
  operand_words<TYPE>(y, q);
#pragma unroll
  for (int i = 0; i < PLANES<TYPE>; ++i) {
    const v4u_t w = join_pair(p[i], q[i]);
    if (in) *(gv4u_a16*)((uint16_t*)base + at + i * plane) = w;
  }
}

// a and b of one fragment, four of either a lane.  16-bit types: 16 bytes of
// upper halves a lane, then, behind all fragments', 8 bytes of the next 8 bits.
template <int TYPE>
__host__ __device__ constexpr int64_t ab_bytes(int64_t fi, int64_t fj) {
  return fi * fj * 64 * (TYPE == SCAO_F32 ? 32 : 24);
}
typedef __attribute__((address_space(1))) v2u gv2u_a8;

template <int TYPE>
__device__ __forceinline__ void put_ab(void* ab, int64_t frags, int64_t frag, int lane, v4f a,
                                       v4f b) {
  const int64_t at = frag * 64 + lane;
  v4u_t ua = __builtin_bit_cast(v4u_t, a), ub = __builtin_bit_cast(v4u_t, b);
  if (TYPE == SCAO_F32) {
    ((gv4u_a16*)ab)[2 * at] = ua;
    ((gv4u_a16*)ab)[2 * at + 1] = ub;
    return;
  }
  v4u_t hi;
  v2u lo;
  // byte selectors of v_perm_b32: 0-3 of the second word, 4-7 of the first
  hi[0] = __builtin_amdgcn_perm(ua[1], ua[0], 0x07060302u);
  hi[1] = __builtin_amdgcn_perm(ua[3], ua[2], 0x07060302u);
  hi[2] = __builtin_amdgcn_perm(ub[1], ub[0], 0x07060302u);
  hi[3] = __builtin_amdgcn_perm(ub[3], ub[2], 0x07060302u);
  lo[0] = __builtin_amdgcn_perm(ua[1], ua[0], 0x0c0c0501u) |
          __builtin_amdgcn_perm(ua[3], ua[2], 0x05010c0cu);
  lo[1] = __builtin_amdgcn_perm(ub[1], ub[0], 0x0c0c0501u) |
          __builtin_amdgcn_perm(ub[3], ub[2], 0x05010c0cu);
  ((gv4u_a16*)ab)[at] = hi;
  ((gv2u_a8*)((char*)ab + frags * 1024))[at] = lo;
}
template <int TYPE>
struct Kept {
  v4u_t hi;   // fp32: a
  v4u_t lo;   // fp32: b; else two words
  __device__ __forceinline__ void load(const void* ab, int64_t frags, int64_t frag, int lane) {
    const int64_t at = frag * 64 + lane;
    if (TYPE == SCAO_F32) {
      hi = ((const gv4u_a16*)ab)[2 * at];
      lo = ((const gv4u_a16*)ab)[2 * at + 1];
    } else {
      hi = ((const gv4u_a16*)ab)[at];
      const v2u w = ((const gv2u_a8*)((const char*)ab + frags * 1024))[at];
      lo[0] = w[0];
      lo[1] = w[1];
    }
  }
  __device__ __forceinline__ void get(v4f& a, v4f& b) const {
    if (TYPE == SCAO_F32) {
      a = __builtin_bit_cast(v4f, hi);
      b = __builtin_bit_cast(v4f, lo);
      return;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      // bytes 1 (from lo), 2 and 3 (from hi) of the float; byte 0 is zero
      const uint32_t half = t & 1 ? 0x0706000cu : 0x0504000cu;
      a[t] = __uint_as_float(__builtin_amdgcn_perm(hi[t / 2], lo[0], half | (uint32_t)t << 8));
      b[t] = __uint_as_float(__builtin_amdgcn_perm(hi[2 + t / 2], lo[1], half | (uint32_t)t << 8));
    }
  }
};

// ------------------------------------------------------ epilogues ----------
// Four consecutive columns n .. n+3 of row m of C.
template <int TYPE>
__device__ __forceinline__ void epi_store(const FfnEpilogue& e, int m, int n, v4f c) {
  void* out = e.out;
  if (m >= e.second) {
    m -= e.second;
    out = e.out2;
  }
  if (m >= e.rows || n >= e.cols || !out) return;
  const int64_t at = (int64_t)m * e.ldo + n;
  const int left = e.cols - n;
  st4(out, TYPE, at, c, left >= 4, left >= 4 ? 15 : (1 << left) - 1);
}

// the same of two fragments next to each other, the first at column n
template <int TYPE>
__device__ __forceinline__ void epi_store_pair(const FfnEpilogue& e, int m, int n, int lane, v4f c,
                                               v4f d) {
  if (TYPE == SCAO_F32) {
    n += 4 * (lane >> 4);
    epi_store<TYPE>(e, m, n, c);
    epi_store<TYPE>(e, m, n + 16, d);
    return;
  }
  v2u p[1], q[1];
  operand_words<TYPE == SCAO_F32 ? SCAO_BF16 : TYPE>(c, p);
  operand_words<TYPE == SCAO_F32 ? SCAO_BF16 : TYPE>(d, q);
  const v4u_t w = join_pair(p[0], q[0]);
  n += pair_column(lane);
  void* out = e.out;
  if (m >= e.second) {
    m -= e.second;
    out = e.out2;
  }
  if (m >= e.rows || n >= e.cols || !out) return;
  uint16_t* to = (uint16_t*)out + (int64_t)m * e.ldo + n;
  if (n + 8 <= e.cols) {
    *(gv4u_a2*)to = w;
  } else {
#pragma unroll
    for (int t = 0; t < 8; ++t)
      if (n + t < e.cols) ((gu16*)to)[t] = (uint16_t)(w[t / 2] >> (16 * (t & 1)));
  }
}

// h of a fragment, a and b kept
template <int TYPE, int ACT>
__device__ __forceinline__ v4f epi_gated(const FfnEpilogue& e, int m, int n, int lane, v4f a,
                                         v4f b) {
  v4f h;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    float f, g;
    activation<ACT, TYPE == SCAO_F32>(a[t], f, g);
    h[t] = f * b[t];
  }
  const int fi = m >> 4, fj = n >> 4;
  if (e.ab && fi < e.fi && fj < e.fj)
    put_ab<TYPE>(e.ab, (int64_t)e.fi * e.fj, (int64_t)fi * e.fj + fj, lane, a, b);
  return h;
}

// where a fragment's a and b are kept; one outside of what is kept repeats the
// last one and writes nothing
__device__ __forceinline__ int64_t kept_at(const FfnEpilogue& e, int m, int n) {
  return (int64_t)min(m >> 4, e.fi - 1) * e.fj + min(n >> 4, e.fj - 1);
}
template <int TYPE, int ACT>
__device__ __forceinline__ void epi_dact(const Kept<TYPE>& k, v4f dh, v4f& da, v4f& db) {
  v4f a, b;
  k.get(a, b);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    float f, g;
    activation<ACT, TYPE == SCAO_F32>(a[t], f, g);
    da[t] = dh[t] * b[t] * g;
    db[t] = dh[t] * f;
  }
}

// f with the activation as a type, chosen outside of the unrolled loops
template <int ACT>
struct Activation {
  static constexpr int value = ACT;
};
template <class F>
__device__ __forceinline__ void for_activation(int act, F&& f) {
  switch (act) {
    case SCAO_ACT_SILU: f(Activation<SCAO_ACT_SILU>{}); break;
    case SCAO_ACT_GELU: f(Activation<SCAO_ACT_GELU>{}); break;
    case SCAO_ACT_GELU_TANH: f(Activation<SCAO_ACT_GELU_TANH>{}); break;
    case SCAO_ACT_RELU: f(Activation<SCAO_ACT_RELU>{}); break;
    default: f(Activation<SCAO_ACT_SIGMOID>{}); break;
  }
}

// ------------------------------------------------------- products ----------
typedef __attribute__((address_space(1))) v4f gv4f_a16;

// Workgroup `block` of one product: a tile, or one part of its k steps.
template <class G, int TYPE, int EPI>
__device__ __forceinline__ void ffn_tile(char* smem, const FfnOperands& o, const FfnEpilogue& e,
                                         int block) {
  const bool split = block >= o.whole;
  const int rest = o.tiles() - o.whole;
  const int part = split ? (block - o.whole) / rest : 0;
  const int tile = block - part * rest;
  int tm, tn;
  tile_of(tile, o.tiles_m, o.tiles_n, tm, tn);
  G g(o, (lchar*)smem, tm, tn);
  const int steps = o.nseg * ((o.K + FFN_BK - 1) / FFN_BK);
  const int per = split ? (steps + o.splits - 1) / o.splits : steps;
  v4f acc[G::MI][G::NJ];
  g.run(part * per, min(steps, part * per + per), acc);

  const int lane = g.lane, dm = lane & 15, dn = 4 * (lane >> 4);
  if (split) {   // a part's sums: tile after tile, a tile's fragments in order
    gv4f_a16* to = (gv4f_a16*)e.partial +
                   ((int64_t)part * rest + (tile - o.whole)) * (G::FRAGS * 64) + lane;
#pragma unroll
    for (int i = 0; i < G::MI; ++i)
#pragma unroll
      for (int j = 0; j < G::NJ; ++j)
        to[(g.frag_m(i) / 16 * (G::BN_ / 16) + g.frag_n(j) / 16) * 64] = acc[i][j];
    return;
  }
  // pairs of fragments next to each other where a wave has them
  constexpr int NH = EPI == EPI_GATED ? G::NJ / 2 : G::NJ, STEP = NH % 2 ? 1 : 2;
  const int dp = STEP == 2 ? pair_column(lane) : dn;
  if constexpr (EPI == EPI_STORE) {
#pragma unroll
    for (int i = 0; i < G::MI; ++i)
#pragma unroll
      for (int j = 0; j < NH; j += STEP) {
        const int m = g.m0 + g.frag_m(i) + dm, n = g.n0 + g.frag_n(j);
        if constexpr (STEP == 2) epi_store_pair<TYPE>(e, m, n, lane, acc[i][j], acc[i][j + 1]);
        else epi_store<TYPE>(e, m, n + dn, acc[i][j]);
      }
  } else if constexpr (EPI == EPI_GATED) {
    auto epilogue = [&](auto act) __attribute__((always_inline)) {
      constexpr int ACT = decltype(act)::value;
#pragma unroll
      for (int i = 0; i < G::MI; ++i)
#pragma unroll
        for (int j = 0; j < NH; j += STEP) {
          const int m = g.m0 + g.frag_m(i) + dm, n = g.n0 + g.frag_n(j);
          const v4f h = epi_gated<TYPE, ACT>(e, m, n + dn, lane, acc[i][j], acc[i][j + NH]);
          const bool in = m < e.rows && n + dp < e.cols;
          const int64_t at = (int64_t)m * e.ldo + n + dp;
          if constexpr (STEP == 2)
            put_operand_pair<TYPE>(e.out, at, e.plane, in, h,
                                   epi_gated<TYPE, ACT>(e, m, n + 16 + dn, lane, acc[i][j + 1],
                                                        acc[i][j + 1 + NH]));
          else if (in) put_operand<TYPE>(e.out, at, e.plane, h);
        }
    };
    for_activation(e.act, epilogue);
  } else {
    // A wait for loads also waits for the stores before them, so the kept values
    // of many fragments are loaded at a time (dh of 4096 tokens x 8192 with k =
    // 64, so nearly the epilogue alone: 123 us one fragment at a time, 83 with
    // 16); more than 8 do not fit beside the 256 x 256 tile's sums.
    auto epilogue = [&](auto act) __attribute__((always_inline)) {
      constexpr int ACT = decltype(act)::value;
      constexpr int BATCH = G::MI * G::NJ > 16 ? 1 : G::MI < 4 ? G::MI : 4;
#pragma unroll
      for (int i0 = 0; i0 < G::MI; i0 += BATCH) {
        Kept<TYPE> k[BATCH][NH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
#pragma unroll
          for (int j = 0; j < NH; ++j)
            k[i][j].load(e.ab, (int64_t)e.fi * e.fj,
                         kept_at(e, g.m0 + g.frag_m(i0 + i), g.n0 + g.frag_n(j)), lane);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
#pragma unroll
          for (int j = 0; j < NH; j += STEP) {
            __builtin_amdgcn_sched_barrier(0);
            const int m = g.m0 + g.frag_m(i0 + i) + dm, n = g.n0 + g.frag_n(j) + dp;
            const bool in = m < e.rows && n < e.cols;
            const int64_t at = (int64_t)m * e.ldo + n;
            v4f da, db, da2, db2;
            epi_dact<TYPE, ACT>(k[i][j], acc[i0 + i][j], da, db);
            if constexpr (STEP == 2) {
              epi_dact<TYPE, ACT>(k[i][j + 1], acc[i0 + i][j + 1], da2, db2);
              put_operand_pair<TYPE>(e.out, at, e.plane, in, da, da2);
              put_operand_pair<TYPE>(e.out, at + e.ldo / 2, e.plane, in, db, db2);
            } else if (in) {
              put_operand<TYPE>(e.out, at, e.plane, da);
              put_operand<TYPE>(e.out, at + e.ldo / 2, e.plane, db);
            }
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    for_activation(e.act, epilogue);
  }
}

template <class G, int TYPE, int EPI>
__global__ __launch_bounds__(G::THREADS, 2) void k_ffn_gemm(const FfnOperands o,
                                                            const FfnEpilogue e) {
  __shared__ __attribute__((aligned(1024))) char smem[G::LDS];
  ffn_tile<G, TYPE, EPI>(smem, o, e, blockIdx.x);
}

// Two products that do not need each other in one launch: the second one's tiles
// fill the CUs that the first one's last round would leave idle.  na: workgroups
// of the first.  `mixed` eights of either take turns (eight, so that a tile keeps
// its XCD), so that dh's epilogue moves its bytes while other CUs multiply; then
// come the longer tiles' rest and the shorter ones'.
template <class GA, int EPI_A, class GB, int EPI_B, int TYPE>
__global__ __launch_bounds__(GA::THREADS, 2) void k_ffn_pair(const FfnOperands oa,
                                                             const FfnEpilogue ea,
                                                             const FfnOperands ob,
                                                             const FfnEpilogue eb, int na, int nb,
                                                             int mixed, int b_leads) {
  static_assert(GA::THREADS == GB::THREADS, "one shape of workgroup");
  __shared__ __attribute__((aligned(1024))) char smem[GA::LDS > GB::LDS ? GA::LDS : GB::LDS];
  int b = blockIdx.x;
  bool lead;
  if (b < 16 * mixed) {
    lead = b / 8 % 2 == 0;
    b = b / 16 * 8 + b % 8;
  } else {
    b -= 8 * mixed;
    const int n = b_leads ? nb : na;
    lead = b < n;
    if (!lead) b -= n - 8 * mixed;
  }
  if (lead != (b_leads != 0)) ffn_tile<GA, TYPE, EPI_A>(smem, oa, ea, b);
  else ffn_tile<GB, TYPE, EPI_B>(smem, ob, eb, b);
}

// The parts of a split product's tiles, added in order, and their epilogue: a
// wave takes a fragment (GATED: one of either projection).  Four parts are under
// way at a time, since few workgroups wait for memory here.
template <class G, int TYPE, int EPI>
__device__ __forceinline__ void ffn_join(const FfnOperands& o, const FfnEpilogue& e, int block) {
  constexpr int FJ = G::COLS_N / 16, FRAGS = G::BM_ / 16 * FJ;   // of C in a tile
  const int64_t frag = (int64_t)block * 4 + (threadIdx.x >> 6);
  const int rest = o.tiles() - o.whole;
  if (frag >= (int64_t)rest * FRAGS) return;
  const int lane = threadIdx.x & 63, tile = (int)(frag / FRAGS), in = (int)(frag % FRAGS);
  int tm, tn;
  tile_of(o.whole + tile, o.tiles_m, o.tiles_n, tm, tn);
  const int m = o.row0 + tm * G::BM_ + in / FJ * 16 + (lane & 15);
  const int n = tn * G::COLS_N + in % FJ * 16 + 4 * (lane >> 4);
  if (m - (lane & 15) >= o.M || n - 4 * (lane >> 4) >= e.cols) return;
  // in the tile's own order of fragments an up fragment follows the gate's row
  const gv4f_a16* p = (const gv4f_a16*)e.partial +
                      ((int64_t)tile * G::FRAGS + in / FJ * (G::BN_ / 16) + in % FJ) * 64 + lane;
  const int64_t all = (int64_t)rest * G::FRAGS * 64;
  Kept<TYPE> k;
  if (EPI == EPI_DACT) k.load(e.ab, (int64_t)e.fi * e.fj, kept_at(e, m, n), lane);
  v4f a = {0.f, 0.f, 0.f, 0.f}, b = a;
  constexpr int BATCH = 4;
  for (int s = 0; s < o.splits; s += BATCH) {
    v4f pa[BATCH], pb[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (s + i < o.splits) {
        pa[i] = p[(s + i) * all];
        if (EPI == EPI_GATED) pb[i] = p[(s + i) * all + FJ * 64];
      }
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (s + i < o.splits) {
        a += pa[i];
        if (EPI == EPI_GATED) b += pb[i];
      }
  }
  if constexpr (EPI == EPI_STORE) {
    epi_store<TYPE>(e, m, n, a);
  } else {
    const bool in = m < e.rows && n < e.cols;
    const int64_t at = (int64_t)m * e.ldo + n;
    for_activation(e.act, [&](auto act) {
      constexpr int ACT = decltype(act)::value;
      if constexpr (EPI == EPI_GATED) {
        const v4f h = epi_gated<TYPE, ACT>(e, m, n, lane, a, b);
        if (in) put_operand<TYPE>(e.out, at, e.plane, h);
      } else {
        v4f da, db;
        epi_dact<TYPE, ACT>(k, a, da, db);
        if (in) {
          put_operand<TYPE>(e.out, at, e.plane, da);
          put_operand<TYPE>(e.out, at + e.ldo / 2, e.plane, db);
        }
      }
    });
  }
}

template <class G, int TYPE, int EPI>
__global__ __launch_bounds__(256) void k_ffn_join(const FfnOperands o, const FfnEpilogue e) {
  ffn_join<G, TYPE, EPI>(o, e, blockIdx.x);
}
// of both products of a pair; na: workgroups of the first's
template <class GA, int EPI_A, class GB, int EPI_B, int TYPE>
__global__ __launch_bounds__(256) void k_ffn_join_pair(const FfnOperands oa, const FfnEpilogue ea,
                                                       const FfnOperands ob, const FfnEpilogue eb,
                                                       int na) {
  if ((int)blockIdx.x < na) ffn_join<GA, TYPE, EPI_A>(oa, ea, blockIdx.x);
  else ffn_join<GB, TYPE, EPI_B>(ob, eb, blockIdx.x - na);
}

// --------------------------------------------------------- packing ---------
// Matrices with any row stride and start as products' operands: rows of `ldo`
// elements (cols rounded up to 8, the rest zero), 16-byte aligned; an fp32 one as
// three bf16 planes that add up to it.  Eight columns a thread; all matrices of a
// pass in one launch.
constexpr int FFN_MAX_PACK = 5;
struct FfnPack {
  struct Matrix {
    const void* src;
    void* dst;
    int64_t ld, plane, rows;
    int cols, ldo;
    int64_t first;          // workgroups before this matrix
  } m[FFN_MAX_PACK];
  int n;
  int64_t groups;
};
typedef v4f v4f_a4 __attribute__((aligned(4)));
typedef __attribute__((address_space(1))) v4f_a4 gv4f_a4;
template <int TYPE>
__global__ __launch_bounds__(256) void k_ffn_pack(const FfnPack p) {
  int k = 0;
#pragma unroll
  for (int i = 1; i < FFN_MAX_PACK; ++i)
    if (i < p.n && (int64_t)blockIdx.x >= p.m[i].first) k = i;
  const FfnPack::Matrix& m = p.m[k];
  const int per = m.ldo / 8;
  const int64_t i0 = ((int64_t)blockIdx.x - m.first) * 256;
  const int at = (int)(i0 % per) + threadIdx.x;
  const int64_t r = i0 / per + at / per;
  if (r >= m.rows) return;
  const int c = at % per * 8, left = m.cols - c;
  uint16_t* dst = (uint16_t*)m.dst + r * m.ldo + c;
  if constexpr (TYPE == SCAO_F32) {
    const gfloat* src = (const gfloat*)m.src + r * m.ld + c;
    v4f x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    if (left >= 8) {
      x[0] = ((const gv4f_a4*)src)[0];
      x[1] = ((const gv4f_a4*)src)[1];
    } else {
#pragma unroll
      for (int t = 0; t < 8; ++t)
        if (t < left) x[t / 4][t % 4] = src[t];
    }
    v2u w[2][3];
    operand_words<SCAO_F32>(x[0], w[0]);
    operand_words<SCAO_F32>(x[1], w[1]);
#pragma unroll
    for (int i = 0; i < 3; ++i)
      *(gv4u_a16*)(dst + i * m.plane) = v4u_t{w[0][i][0], w[0][i][1], w[1][i][0], w[1][i][1]};
  } else {
    const gu16* src = (const gu16*)m.src + r * m.ld + c;
    v4u_t w = {0, 0, 0, 0};
    if (left >= 8) {
      w = *(const gv4u_a2*)src;
    } else {
#pragma unroll
      for (int t = 0; t < 8; ++t)
        if (t < left) w[t / 2] |= (uint32_t)src[t] << (16 * (t % 2));
    }
    *(gv4u_a16*)dst = w;
  }
}

// --------------------------------------------------------- launches --------
// The products by the layouts of their operands and their epilogue.
enum { FFN_GATE_UP, FFN_DOWN, FFN_DH, FFN_DX, FFN_DW };

// The tiles, and how many columns of C one covers: half of BN for GATE_UP.  256 x
// 128 is for DOWN.
enum { FFN_256x256, FFN_256x128, FFN_128x128, FFN_64x128, FFN_32x128, FFN_TILES };
constexpr int FFN_BM[FFN_TILES] = {256, 256, 128, 64, 32};
constexpr int FFN_BN[FFN_TILES] = {256, 128, 128, 128, 128};

template <int TYPE, int TILE, int WM, int WN, int LA, int LB, int EPI>
using FfnTile =
    Gemm<FFN_BM[TILE], FFN_BN[TILE], WM, WN, LA, LB, TYPE == SCAO_F16, EPI == EPI_GATED>;

template <class G>
int join_groups(const FfnOperands& o) {
  const int64_t frags = (int64_t)(o.tiles() - o.whole) * (G::BM_ / 16) * (G::COLS_N / 16);
  return (int)((frags + 3) / 4);
}
template <class G, int TYPE, int EPI>
void launch_join(const FfnOperands& o, const FfnEpilogue& e, hipStream_t st) {
  if (const int n = join_groups<G>(o)) k_ffn_join<G, TYPE, EPI><<<n, 256, 0, st>>>(o, e);
}

template <int TYPE, int TILE, int WM, int WN, int LA, int LB, int EPI>
void launch_gemm(const FfnOperands& o, const FfnEpilogue& e, hipStream_t st) {
  using G = FfnTile<TYPE, TILE, WM, WN, LA, LB, EPI>;
  k_ffn_gemm<G, TYPE, EPI><<<o.groups(), G::THREADS, 0, st>>>(o, e);
  launch_join<G, TYPE, EPI>(o, e, st);
}

// the products of the backward pass that go together: dh or dx, and a dW
template <int TYPE, int TILE, int WM, int WN, int EPI>
void launch_pair_tile(const FfnOperands& oa, const FfnEpilogue& ea, const FfnOperands& ob,
                      const FfnEpilogue& eb, hipStream_t st) {
  using A = FfnTile<TYPE, TILE, WM, WN, ROWS, COLS, EPI>;
  using B = FfnTile<TYPE, TILE, WM, WN, COLS, COLS, EPI_STORE>;
  const int na = oa.groups(), nb = ob.groups();
  const int mixed = EPI == EPI_DACT ? (na < nb ? na : nb) / 8 : 0;
  const int64_t sa = (int64_t)oa.nseg * ((oa.K + FFN_BK - 1) / FFN_BK) / oa.splits;
  const int64_t sb = (int64_t)ob.nseg * ((ob.K + FFN_BK - 1) / FFN_BK) / ob.splits;
  k_ffn_pair<A, EPI, B, EPI_STORE, TYPE>
      <<<na + nb, A::THREADS, 0, st>>>(oa, ea, ob, eb, na, nb, mixed, sb > sa);
  const int ja = join_groups<A>(oa), jb = join_groups<B>(ob);
  if (ja && jb)
    k_ffn_join_pair<A, EPI, B, EPI_STORE, TYPE><<<ja + jb, 256, 0, st>>>(oa, ea, ob, eb, ja);
  else if (ja)
    k_ffn_join<A, TYPE, EPI><<<ja, 256, 0, st>>>(oa, ea);
  else if (jb)
    k_ffn_join<B, TYPE, EPI_STORE><<<jb, 256, 0, st>>>(ob, eb);
}
template <int TYPE>
void launch_pair(int kind, int tile, const FfnOperands& oa, const FfnEpilogue& ea,
                 const FfnOperands& ob, const FfnEpilogue& eb, hipStream_t st) {
  if (kind == FFN_DH) {
    if (tile == FFN_256x256) launch_pair_tile<TYPE, FFN_256x256, 2, 4, EPI_DACT>(oa, ea, ob, eb, st);
    else launch_pair_tile<TYPE, FFN_128x128, 2, 2, EPI_DACT>(oa, ea, ob, eb, st);
  } else {
    if (tile == FFN_256x256)
      launch_pair_tile<TYPE, FFN_256x256, 2, 4, EPI_STORE>(oa, ea, ob, eb, st);
    else launch_pair_tile<TYPE, FFN_128x128, 2, 2, EPI_STORE>(oa, ea, ob, eb, st);
  }
}

template <int TYPE, int LA, int LB, int EPI>
void launch_tile(int tile, const FfnOperands& o, const FfnEpilogue& e, hipStream_t st) {
  if (tile == FFN_256x256) launch_gemm<TYPE, FFN_256x256, 2, 4, LA, LB, EPI>(o, e, st);
  else if (tile == FFN_128x128) launch_gemm<TYPE, FFN_128x128, 2, 2, LA, LB, EPI>(o, e, st);
  if constexpr (LA == ROWS) {   // A's rows are tokens: there may be few
    if (tile == FFN_64x128) launch_gemm<TYPE, FFN_64x128, 1, 4, LA, LB, EPI>(o, e, st);
    else if (tile == FFN_32x128) launch_gemm<TYPE, FFN_32x128, 1, 4, LA, LB, EPI>(o, e, st);
    if constexpr (LB == ROWS && EPI == EPI_STORE)
      if (tile == FFN_256x128) launch_gemm<TYPE, FFN_256x128, 4, 2, LA, LB, EPI>(o, e, st);
  }
}

template <int TYPE>
void launch_product(int kind, int tile, const FfnOperands& o, const FfnEpilogue& e,
                    hipStream_t st) {
  switch (kind) {
    case FFN_GATE_UP: launch_tile<TYPE, ROWS, ROWS, EPI_GATED>(tile, o, e, st); break;
    case FFN_DOWN: launch_tile<TYPE, ROWS, ROWS, EPI_STORE>(tile, o, e, st); break;
    case FFN_DH: launch_tile<TYPE, ROWS, COLS, EPI_DACT>(tile, o, e, st); break;
    case FFN_DX: launch_tile<TYPE, ROWS, COLS, EPI_STORE>(tile, o, e, st); break;
    default: launch_tile<TYPE, COLS, COLS, EPI_STORE>(tile, o, e, st); break;
  }
}

template <int TYPE>
void launch_pack(const FfnPack& p, hipStream_t st) {
  k_ffn_pack<TYPE><<<(int)p.groups, 256, 0, st>>>(p);
}

struct FfnFew;
// instantiated in ffn_f32.hip, ffn_bf16.hip and ffn_f16.hip
struct FfnLaunchers {
  void (*product)(int, int, const FfnOperands&, const FfnEpilogue&, hipStream_t);
  void (*pair)(int, int, const FfnOperands&, const FfnEpilogue&, const FfnOperands&,
               const FfnEpilogue&, hipStream_t);
  void (*pack)(const FfnPack&, hipStream_t);
  void (*few)(const FfnFew&, const FfnEpilogue&, bool, hipStream_t);
};
FfnLaunchers ffn_f32();
FfnLaunchers ffn_bf16();
FfnLaunchers ffn_f16();

}  // namespace scao
