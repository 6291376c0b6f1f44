// Norms of queries and keys for each head with the rotation by the token's position
// in the same pass, and its backward pass, on gfx950.
//
//   r = 1 / sqrt(mean x^2 + eps), u = r x, y = u w
//   y'_i = y_i cos - y_j sin, y'_j = y_j cos + y_i sin       for the pairs (i, j)
// backward, with dy = dy' rotated back:
//   dw = sum dy u, du = dy w, dx = r (du - u mean(du u))
//
// Everything follows from x, so the forward pass keeps nothing.  Sums and products
// are fp32, outputs rounded once.
//
// A head's columns are walked in pairs of pieces of V elements (16 bytes): piece c of
// the first half beside piece c of the second, whose elements rotate together (pairs
// half a rotation apart), or two pieces side by side (pairs next to each other); the
// columns behind the rotated ones follow as pairs of pieces that do not rotate.  A lane
// holds one such pair, L lanes a head, so that a rotation needs no other lane and a
// mean log2 L exchanges.  V is 8 or 4 and less where the head's or the rotation's size
// asks for it, down to single elements.
//
// Bound by HBM: 8192 tokens of 32 + 8 heads of 128 in bf16, forward 34 us (4.9 TB/s),
// backward 54 and its join 5 (4.7 TB/s); by the launch for few tokens (one: 5 us).  In
// the forward pass a group of L lanes takes four heads of one token: the token's cosines
// and sines, twice the bytes of a head's 16-bit data, are read once for all of them, and
// four heads' loads are under way (two: 35 us; pieces of 8 bytes: 37).
#include <algorithm>

#include "../../include/scao_train.h"
#include "scao_common.hpp"

using namespace scao;

namespace {

int size_of(int dt) { return dt == SCAO_F32 ? 4 : 2; }

constexpr int THREADS = 256;
constexpr int MAX_DIM = 512;
constexpr int MAX_BLOCKS = 768;     // of a backward pass, with a partial sum each

// one of the two tensors
struct Side {
  const void* x;
  const void* w;             // or null: ones
  const void* dy;
  void* out;                 // y' or dx; null: not wanted
  int64_t xb, xt, xh;        // strides of batch, token and head, in elements
  int64_t yb, yt, yh;        // of dy
  int64_t ob, ot, oh;        // of out
  int heads, runs, w_dtype;  // runs of heads that one group takes
};
struct Args {
  Side s[2];
  const float* cos;
  const float* sin;
  const void* positions;     // or null: the token's place in its sequence
  float* parts;              // backward: the workgroups' sums for both weights, or null
  int64_t ld_table, pb, pt;  // strides of the tables' rows and of positions
  uint32_t tokens, seq;
  int64_t table;             // rows of the tables
  int dim, half;             // columns; half the rotated ones
  int wide_positions;
  int lanes;                 // of a head
  float eps;
};

typedef __attribute__((address_space(1))) const int64_t gi64;
typedef __attribute__((address_space(1))) const int32_t gi32;
typedef uint32_t v1u_a2 __attribute__((aligned(2)));
typedef v4u_t v4u_a2 __attribute__((aligned(2)));
typedef float v2f_a4 __attribute__((ext_vector_type(2), aligned(4)));
#define GLOBAL(T) __attribute__((address_space(1))) T

// V elements in a row, which start at any element: as they are in memory, and as
// numbers.  (They are held as they are until they are needed.)
template <int DT, int V>
struct Words {
  static constexpr int N = DT == SCAO_F32 ? V : V > 1 ? V / 2 : 1;
  uint32_t w[N];
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    if constexpr (DT == SCAO_F32) {
      if constexpr (V == 1) {
        w[0] = __float_as_uint(gld1((const float*)p + at));
      } else if constexpr (V == 2) {
        const v2f_a4 v = *(const GLOBAL(v2f_a4)*)((const float*)p + at);
        w[0] = __float_as_uint(v[0]);
        w[1] = __float_as_uint(v[1]);
      } else {
#pragma unroll
        for (int h = 0; h < V; h += 4) {
          const v4f v = gld4((const float*)p + at + h);
#pragma unroll
          for (int t = 0; t < 4; ++t) w[h + t] = __float_as_uint(v[t]);
        }
      }
    } else if constexpr (V == 1) {
      w[0] = ((const gu16*)p)[at];
    } else if constexpr (V == 2) {
      w[0] = *(const GLOBAL(v1u_a2)*)((const uint16_t*)p + at);
    } else if constexpr (V == 4) {
      const v2u v = gld2w((const uint16_t*)p + at);
      w[0] = v[0];
      w[1] = v[1];
    } else {
      const v4u_t v = *(const GLOBAL(v4u_a2)*)((const uint16_t*)p + at);
#pragma unroll
      for (int t = 0; t < 4; ++t) w[t] = v[t];
    }
  }
  __device__ __forceinline__ void get(float (&x)[V]) const {
#pragma unroll
    for (int t = 0; t < V; ++t) {
      if (DT == SCAO_F32)
        x[t] = __uint_as_float(w[t % N]);
      else if (DT == SCAO_BF16)
        x[t] = __uint_as_float(t & 1 ? w[t / 2] & 0xffff0000u : w[t / 2] << 16);
      else
        x[t] = f16_to_f((uint16_t)(w[t / 2] >> (16 * (t & 1))));
    }
  }
};
template <int DT, int V>
__device__ __forceinline__ void load(const void* p, int64_t at, float (&x)[V]) {
  Words<DT, V> w;
  w.load(p, at);
  w.get(x);
}
template <int DT, int V>
__device__ __forceinline__ void store(void* p, int64_t at, const float (&x)[V]) {
  if constexpr (V == 1) {
    st1(p, DT, at, x[0]);
  } else if constexpr (DT == SCAO_F32) {
    if constexpr (V == 2) *(GLOBAL(v2f_a4)*)((float*)p + at) = v2f_a4{x[0], x[1]};
    else gst4((float*)p + at, v4f{x[0], x[1], x[2], x[3]});
  } else {
    uint32_t w[V / 2];
#pragma unroll
    for (int t = 0; t < V / 2; ++t)
      w[t] = DT == SCAO_BF16
                 ? pk_bf16(x[2 * t], x[2 * t + 1])
                 : (uint32_t)f_to_f16(x[2 * t]) | (uint32_t)f_to_f16(x[2 * t + 1]) << 16;
    if constexpr (V == 2) *(GLOBAL(v1u_a2)*)((uint16_t*)p + at) = w[0];
    else if constexpr (V == 4) *(gv2u*)((uint16_t*)p + at) = v2u{w[0], w[1]};
    else *(GLOBAL(v4u_a2)*)((uint16_t*)p + at) = v4u_t{w[0], w[1], w[2], w[3]};
  }
}

// pairs of pieces a lane holds: a head has up to MAX_DIM / 2V, a wave 64 lanes
template <int V>
constexpr int PAIRS = V >= 4 ? 1 : 4 / V;

// The pairs of one lane of a head.  BESIDE: those that turn are next to each other.
template <int DT, int V, bool BESIDE>
struct Lane {
  static constexpr int N = PAIRS<V>;
  int at[N][2];              // column of either piece, -1: none
  bool turns[N];
  float w[N][2][V], cos[N][V], sin[N][V];

  __device__ __forceinline__ Lane(const Args& a, int lane) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int c = lane + 64 * k, rotated = a.half / V;   // pairs that turn
      turns[k] = c < rotated;
      if (BESIDE || !turns[k]) {
        at[k][0] = 2 * c * V;
        at[k][1] = at[k][0] + V;
      } else {
        at[k][0] = c * V;
        at[k][1] = a.half + c * V;
      }
      if (at[k][0] >= a.dim) at[k][0] = -1;
      if (at[k][0] < 0 || at[k][1] >= a.dim) at[k][1] = -1;
    }
  }
  __device__ __forceinline__ void weights(const Side& s) {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int t = 0; t < V; ++t) w[k][h][t] = 1.f;
        if (!s.w || at[k][h] < 0) continue;
        if (s.w_dtype == SCAO_F32) load<SCAO_F32, V>(s.w, at[k][h], w[k][h]);
        else if (s.w_dtype == SCAO_BF16) load<SCAO_BF16, V>(s.w, at[k][h], w[k][h]);
        else load<SCAO_F16, V>(s.w, at[k][h], w[k][h]);
      }
  }
  // those of position p; one outside of the tables: NaN
  __device__ __forceinline__ void angles(const Args& a, int64_t p) {
    const bool in = p >= 0 && p < a.table;
    const int64_t row = in ? p * a.ld_table : 0;
#pragma unroll
    for (int k = 0; k < N; ++k) {
#pragma unroll
      for (int t = 0; t < V; ++t) {
        cos[k][t] = in ? 1.f : __uint_as_float(0x7fc00000u);
        sin[k][t] = 0.f;
      }
      if (turns[k] && in) {
        const int64_t c = row + at[k][0] / (BESIDE ? 2 : 1);
        load<SCAO_F32, V>(a.cos, c, cos[k]);
        load<SCAO_F32, V>(a.sin, c, sin[k]);
      }
    }
  }
  using Head = Words<DT, V>[N][2];
  __device__ __forceinline__ void fetch(const void* p, int64_t head, Head& x) const {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int t = 0; t < Words<DT, V>::N; ++t) x[k][h].w[t] = 0;
        if (at[k][h] >= 0) x[k][h].load(p, head + at[k][h]);
      }
  }
  static __device__ __forceinline__ void get(const Head& w, float (&x)[N][2][V]) {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) w[k][h].get(x[k][h]);
  }
  __device__ __forceinline__ void put(void* p, int64_t head, const float (&x)[N][2][V]) const {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (at[k][h] >= 0) store<DT, V>(p, head + at[k][h], x[k][h]);
  }
  // by the angles, or (BACK) by their negatives
  template <bool BACK>
  static __device__ __forceinline__ void turn(float& p, float& q, float c, float sine) {
    const float s = BACK ? -sine : sine, u = p, v = q;
    p = fmaf(u, c, -(v * s));
    q = fmaf(v, c, u * s);
  }
  // (which columns are pairs is known where this is compiled: chosen by a branch, the
  // values would be held in memory)
  template <bool BACK>
  __device__ __forceinline__ void rotate(float (&x)[N][2][V]) const {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (!turns[k]) continue;
      if (BESIDE) {   // elements 2t and 2t + 1 of both pieces' 2V
#pragma unroll
        for (int t = 0; t < V; ++t)
          turn<BACK>(x[k][2 * t / V][2 * t % V], x[k][(2 * t + 1) / V][(2 * t + 1) % V], cos[k][t],
                     sin[k][t]);
      } else {
#pragma unroll
        for (int t = 0; t < V; ++t) turn<BACK>(x[k][0][t], x[k][1][t], cos[k][t], sin[k][t]);
      }
    }
  }
};

// the position of token t of sequence b
__device__ __forceinline__ int64_t position_of(const Args& a, uint32_t b, uint32_t t) {
  if (!a.positions) return t;
  const int64_t i = b * a.pb + t * a.pt;
  return a.wide_positions ? ((gi64*)a.positions)[i] : ((gi32*)a.positions)[i];
}
// of a head's lanes
__device__ __forceinline__ float over_lanes(float x, int lanes) {
  for (int o = lanes / 2; o > 0; o >>= 1) x += __shfl_xor(x, o, SCAO_WAVE);
  return x;
}

// one side or the other, field by field: two lanes of a wave may differ
__device__ __forceinline__ Side side_of(const Args& a, int side) {
  Side s;
#define PICK(f) s.f = side ? a.s[1].f : a.s[0].f
  PICK(x); PICK(w); PICK(dy); PICK(out);
  PICK(xb); PICK(xt); PICK(xh); PICK(yb); PICK(yt); PICK(yh); PICK(ob); PICK(ot); PICK(oh);
  PICK(heads); PICK(runs); PICK(w_dtype);
#undef PICK
  return s;
}
// run `run` of a token's runs: which side, and its heads
struct Run {
  int side, head, heads;
};
template <int R>
__device__ __forceinline__ Run run_of(const Args& a, int run) {
  const int side = run >= a.s[0].runs, first = (run - side * a.s[0].runs) * R;
  return Run{side, first, min(R, (side ? a.s[1].heads : a.s[0].heads) - first)};
}

constexpr int FORWARD_HEADS = 4;    // under way at a time
template <int DT, int V, bool BESIDE>
__global__ __launch_bounds__(THREADS) void k_rope_forward(const Args a) {
  constexpr int N = PAIRS<V>, R = FORWARD_HEADS;
  const uint32_t group = blockIdx.x * (THREADS / a.lanes) + threadIdx.x / a.lanes;
  const int lane = threadIdx.x & (a.lanes - 1), runs = a.s[0].runs + a.s[1].runs;
  uint32_t token = group / runs;
  Run run = run_of<R>(a, group % runs);
  if (token >= a.tokens) {   // (its lanes take part in the exchanges)
    token = 0;
    run.heads = 0;
  }
  const Side s = side_of(a, run.side);
  const uint32_t b = token / a.seq, t = token % a.seq;
  Lane<DT, V, BESIDE> l(a, lane);
  const int64_t xs = b * s.xb + t * s.xt + run.head * s.xh;
  typename Lane<DT, V, BESIDE>::Head heads[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (r < run.heads) l.fetch(s.x, xs + r * s.xh, heads[r]);
  l.weights(s);
  l.angles(a, position_of(a, b, t));
  const int64_t os = b * s.ob + t * s.ot + run.head * s.oh;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float x[N][2][V], sum = 0.f;
    if (r < run.heads) {
      l.get(heads[r], x);
#pragma unroll
      for (int k = 0; k < N; ++k)
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) sum = fmaf(x[k][e / V][e % V], x[k][e / V][e % V], sum);
    }
    sum = over_lanes(sum, a.lanes);
    const float rms = 1.f / sqrtf(sum / a.dim + a.eps);
    if (r >= run.heads) continue;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) {
        float& y = x[k][e / V][e % V];
        y = y * rms * l.w[k][e / V][e % V];
      }
    l.template rotate<false>(x);
    l.put(s.out, os + r * s.oh, x);
  }
}

// A group keeps its head from token to token, so that a lane adds up its columns of
// one weight's gradient; a workgroup's groups are added in order.  The next token's
// head and position are under way, as they are in memory, while one is worked on: 8192
// tokens of 32 + 8 heads of 128 in bf16 54 us (4.7 TB/s); with two heads a group 55 on
// two thirds of the waves and 111 on as many (registers), without the next head 76.
constexpr int BACKWARD_HEADS = 1;
template <int DT, int V, bool BESIDE>
__global__ __launch_bounds__(THREADS, 3) void k_rope_backward(const Args a) {
  constexpr int N = PAIRS<V>;
  __shared__ float sums[THREADS * 2 * V * N];
  const int groups = THREADS / a.lanes, own = threadIdx.x / a.lanes;
  const int lane = threadIdx.x & (a.lanes - 1), runs = a.s[0].runs + a.s[1].runs;
  const uint32_t group = blockIdx.x * groups + own, tracks = gridDim.x * groups / runs;
  uint32_t token = group / runs;
  const Run run = run_of<BACKWARD_HEADS>(a, group % runs);
  const Side s = side_of(a, run.side);
  if (token >= tracks) token = a.tokens;   // none: the last few groups
  Lane<DT, V, BESIDE> l(a, lane);
  l.weights(s);
  float dw[N][2][V];
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) dw[k][e / V][e % V] = 0.f;

  typename Lane<DT, V, BESIDE>::Head xn = {}, dn = {};
  int64_t position = 0, on = 0;   // and where dx goes
  auto begin = [&](uint32_t i) {
    if (i >= a.tokens) return;
    const uint32_t b = i / a.seq, t = i % a.seq;
    position = position_of(a, b, t);
    l.fetch(s.x, b * s.xb + t * s.xt + run.head * s.xh, xn);
    l.fetch(s.dy, b * s.yb + t * s.yt + run.head * s.yh, dn);
    on = b * s.ob + t * s.ot + run.head * s.oh;
  };
  begin(token);
  // (every lane goes round as often as the one with the most tokens)
  const uint32_t rounds = (a.tokens + tracks - 1) / tracks;
  for (uint32_t i = 0; i < rounds; ++i, token += tracks) {
    const bool in = token < a.tokens;
    const int64_t os = on;
    float x[N][2][V], d[N][2][V], square = 0.f, product = 0.f;
    if (in) {
      l.angles(a, position);
      l.get(xn, x);
      l.get(dn, d);
      begin(token + tracks);
      l.template rotate<true>(d);
#pragma unroll
      for (int k = 0; k < N; ++k)
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) {
          const float v = x[k][e / V][e % V];
          square = fmaf(v, v, square);
          product = fmaf(d[k][e / V][e % V] * l.w[k][e / V][e % V], v, product);
        }
    }
    square = over_lanes(square, a.lanes);
    product = over_lanes(product, a.lanes);
    if (!in) continue;
    const float rms = 1.f / sqrtf(square / a.dim + a.eps);
    const float mean = product * rms / a.dim;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) {
        const float u = x[k][e / V][e % V] * rms, g = d[k][e / V][e % V];
        dw[k][e / V][e % V] = fmaf(g, u, dw[k][e / V][e % V]);
        x[k][e / V][e % V] = rms * fmaf(-u, mean, g * l.w[k][e / V][e % V]);
      }
    if (s.out) l.put(s.out, os, x);
  }
  if (!a.parts) return;
  // [group][column]: dim columns of lanes * 2 V N at most
  const int width = a.lanes * 2 * V * N;
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (l.at[k][h] >= 0)
#pragma unroll
        for (int t = 0; t < V; ++t) sums[own * width + l.at[k][h] + t] = dw[k][h][t];
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.dim; i += THREADS) {
    const int side = i >= a.dim, column = i - side * a.dim;
    float x = 0.f;
    for (int g = 0; g < groups; ++g) {
      const int of = (blockIdx.x * groups + g) % runs >= (uint32_t)a.s[0].runs;
      if (of == side) x += sums[g * width + column];
    }
    a.parts[(int64_t)blockIdx.x * 2 * a.dim + i] = x;
  }
}

// The workgroups' sums, added in order in double: 16 columns a workgroup, 64 threads
// a column, each with eight loads under way.
constexpr int JOIN_ROWS = 64;
struct JoinArgs {
  const float* parts;
  void* dw[2];
  int w_dtype[2];
  int blocks, dim;
};
__global__ __launch_bounds__(16 * JOIN_ROWS) void k_rope_join(const JoinArgs a) {
  __shared__ double sums[JOIN_ROWS][17];
  const int c = threadIdx.x % 16, row = threadIdx.x / 16, i = blockIdx.x * 16 + c;
  double x = 0.0;
  constexpr int AHEAD = 8;
  if (i < 2 * a.dim)
    for (int b = row; b < a.blocks; b += JOIN_ROWS * AHEAD) {
      float p[AHEAD];
#pragma unroll
      for (int t = 0; t < AHEAD; ++t)
        p[t] = b + t * JOIN_ROWS < a.blocks
                   ? gld1(a.parts + (int64_t)(b + t * JOIN_ROWS) * 2 * a.dim + i)
                   : 0.f;
#pragma unroll
      for (int t = 0; t < AHEAD; ++t) x += p[t];
    }
  sums[row][c] = x;
  __syncthreads();
  for (int half = JOIN_ROWS / 2; half > 0; half /= 2) {
    if (row < half) sums[row][c] += sums[row + half][c];
    __syncthreads();
  }
  if (row || i >= 2 * a.dim) return;
  const int side = i >= a.dim;
  if (a.dw[side]) st1(a.dw[side], a.w_dtype[side], i - side * a.dim, (float)sums[0][c]);
}

// ------------------------------------------------------------------ host ---
int check(const char* who, const scao_rope_desc* d) {
  SCAO_CHECK_ARG(d, "%s: null descriptor", who);
  SCAO_CHECK_ARG(d->dtype >= 0 && d->dtype <= SCAO_F16, "%s: dtype %d", who, d->dtype);
  SCAO_CHECK_ARG(d->dim >= 1 && d->dim <= MAX_DIM, "%s: head size %d (1 to %d)", who, d->dim, MAX_DIM);
  SCAO_CHECK_ARG(d->rotary >= 0 && d->rotary <= d->dim && d->rotary % 2 == 0,
                 "%s: %d rotated columns of %d", who, d->rotary, d->dim);
  SCAO_CHECK_ARG(d->heads[0] >= 1 && d->heads[1] >= 1 && d->heads[0] < 65536 && d->heads[1] < 65536,
                 "%s: %d and %d heads", who, d->heads[0], d->heads[1]);
  SCAO_CHECK_ARG(d->batch >= 0 && d->seq >= 0 && d->batch < ((int64_t)1 << 31) &&
                     d->seq < ((int64_t)1 << 31) && d->batch * d->seq < ((int64_t)1 << 31) &&
                     // groups of lanes are counted in 32 bits
                     d->batch * d->seq * (((int64_t)d->heads[0] + d->heads[1]) / 2 + 2) <
                         ((int64_t)1 << 31),
                 "%s: %lld sequences of %lld tokens", who, (long long)d->batch, (long long)d->seq);
  SCAO_CHECK_ARG(d->eps >= 0 && d->eps < 3e38f, "%s: eps %g", who, d->eps);
  for (int i = 0; i < 2; ++i)
    SCAO_CHECK_ARG(!d->w[i] || (d->w_dtype[i] >= 0 && d->w_dtype[i] <= SCAO_F16 &&
                                (uintptr_t)d->w[i] % size_of(d->w_dtype[i]) == 0),
                   "%s: weight %d's type or alignment", who, i);
  if (d->rotary) {
    SCAO_CHECK_ARG(d->cos && d->sin && (uintptr_t)d->cos % 4 == 0 && (uintptr_t)d->sin % 4 == 0,
                   "%s: a table is null or not aligned", who);
    SCAO_CHECK_ARG(d->table_rows >= 0 && (d->table_rows <= 1 || d->ld_table >= d->rotary / 2),
                   "%s: tables of %lld rows %lld apart", who, (long long)d->table_rows,
                   (long long)d->ld_table);
  }
  SCAO_CHECK_ARG(!d->positions || (uintptr_t)d->positions % (d->wide_positions ? 8 : 4) == 0,
                 "%s: positions are not aligned", who);
  return SCAO_OK;
}
int check_tensor(const char* who, const char* name, const scao_rope_desc* d,
                 const scao_rope_tensor& t) {
  SCAO_CHECK_ARG(t.p && (uintptr_t)t.p % size_of(d->dtype) == 0,
                 "%s: %s is null or not aligned to its elements", who, name);
  return SCAO_OK;
}

// Elements of a piece: as many as 16 bytes hold where the columns allow it.
int piece_of(const scao_rope_desc& d) {
  for (int v = d.dtype == SCAO_F32 ? 4 : 8; v > 1; v /= 2)
    if (d.dim % v == 0 && d.rotary / 2 % v == 0) return v;
  return 1;
}
Args args_of(const scao_rope_desc& d, int run, int v) {
  Args a{};
  a.cos = d.cos;
  a.sin = d.sin;
  a.positions = d.rotary ? d.positions : nullptr;
  a.ld_table = d.ld_table;
  a.pb = d.position_strides[0];
  a.pt = d.position_strides[1];
  a.tokens = (uint32_t)(d.batch * d.seq);
  a.seq = (uint32_t)d.seq;
  // (nothing turns: no token's position matters)
  a.table = d.rotary ? d.table_rows : (int64_t)1 << 62;
  a.dim = d.dim;
  a.half = d.rotary / 2;
  a.wide_positions = d.wide_positions != 0;
  a.eps = d.eps;
  const int pairs = (d.dim + 2 * v - 1) / (2 * v);   // of pieces
  a.lanes = 1;
  while (a.lanes < pairs && a.lanes < 64) a.lanes *= 2;
  for (int i = 0; i < 2; ++i) {
    Side& s = a.s[i];
    const scao_rope_tensor& x = d.x[i];
    s.x = x.p;
    s.xb = x.batch;
    s.xt = x.token;
    s.xh = x.head;
    s.w = d.w[i];
    s.w_dtype = d.w_dtype[i];
    s.heads = d.heads[i];
    s.runs = (d.heads[i] + run - 1) / run;
  }
  return a;
}
void to_out(Side& s, const scao_rope_tensor& t) {
  s.out = t.p;
  s.ob = t.batch;
  s.ot = t.token;
  s.oh = t.head;
}
void to_dy(Side& s, const scao_rope_tensor& t) {
  s.dy = t.p;
  s.yb = t.batch;
  s.yt = t.token;
  s.yh = t.head;
}

// f(type, elements of a piece, pairs side by side) as compile-time numbers
template <int I>
struct Number {
  static constexpr int value = I;
};
template <class F>
void for_variant(int dt, int v, bool beside, F&& f) {
  auto sized = [&](auto type, auto piece) {
    if (beside) f(type, piece, Number<1>{});
    else f(type, piece, Number<0>{});
  };
  auto typed = [&](auto type) {
    if (v == 1) sized(type, Number<1>{});
    else if (v == 2) sized(type, Number<2>{});
    else if (v == 4) sized(type, Number<4>{});
    else if constexpr (decltype(type)::value != SCAO_F32) sized(type, Number<8>{});
  };
  if (dt == SCAO_F32) typed(Number<SCAO_F32>{});
  else if (dt == SCAO_BF16) typed(Number<SCAO_BF16>{});
  else typed(Number<SCAO_F16>{});
}

int backward_blocks(const Args& a) {
  const int groups = THREADS / a.lanes, runs = a.s[0].runs + a.s[1].runs;
  const int64_t all = ((int64_t)a.tokens * runs + groups - 1) / groups;
  // at least one track of every run, and as many tokens for each
  const int64_t least = (runs + groups - 1) / groups, rounds = (all + MAX_BLOCKS - 1) / MAX_BLOCKS;
  return (int)std::max(least, (all + rounds - 1) / rounds);
}

}  // namespace

extern "C" int scao_qk_rope_forward(const scao_rope_desc* d, const scao_rope_tensor* y,
                                    void* stream) {
  const char* who = "scao_qk_rope_forward";
  if (int rc = check(who, d)) return rc;
  SCAO_CHECK_ARG(y, "%s: null outputs", who);
  if (d->batch * d->seq == 0) return SCAO_OK;
  for (int i = 0; i < 2; ++i) {
    if (int rc = check_tensor(who, i ? "k" : "q", d, d->x[i])) return rc;
    if (int rc = check_tensor(who, i ? "k's output" : "q's output", d, y[i])) return rc;
  }
  const int v = piece_of(*d);
  Args a = args_of(*d, FORWARD_HEADS, v);
  for (int i = 0; i < 2; ++i) to_out(a.s[i], y[i]);
  const int64_t threads = (int64_t)a.tokens * (a.s[0].runs + a.s[1].runs) * a.lanes;
  const int64_t blocks = (threads + THREADS - 1) / THREADS;
  SCAO_CHECK_ARG(blocks * THREADS < (int64_t)1 << 32,
                 "%s: %lld tokens' heads take %lld lanes (below 2^32)", who, (long long)a.tokens,
                 (long long)threads);
  for_variant(d->dtype, v, d->interleaved != 0, [&](auto type, auto piece, auto beside) {
    k_rope_forward<decltype(type)::value, decltype(piece)::value, decltype(beside)::value != 0>
        <<<(uint32_t)blocks, THREADS, 0, (hipStream_t)stream>>>(a);
  });
  SCAO_LAUNCH_CHECK(who);
  return SCAO_OK;
}

extern "C" int64_t scao_qk_rope_backward_workspace(const scao_rope_desc* d) {
  if (check("scao_qk_rope_backward_workspace", d) || d->batch * d->seq == 0) return 0;
  const Args a = args_of(*d, BACKWARD_HEADS, piece_of(*d));
  return (int64_t)backward_blocks(a) * 2 * d->dim * 4;
}

extern "C" int scao_qk_rope_backward(const scao_rope_desc* d, const scao_rope_tensor* dy,
                                     const scao_rope_tensor* dx, void* dw_q, void* dw_k,
                                     void* workspace, void* stream) {
  const char* who = "scao_qk_rope_backward";
  if (int rc = check(who, d)) return rc;
  SCAO_CHECK_ARG(dy && dx, "%s: null gradients", who);
  void* const dw[2] = {dw_q, dw_k};
  for (int i = 0; i < 2; ++i) {
    SCAO_CHECK_ARG(!dw[i] || (d->w[i] && (uintptr_t)dw[i] % size_of(d->w_dtype[i]) == 0),
                   "%s: a gradient without its weight, or not aligned", who);
    SCAO_CHECK_ARG((uintptr_t)dx[i].p % size_of(d->dtype) == 0, "%s: a gradient is not aligned", who);
  }
  JoinArgs j{nullptr, {dw_q, dw_k}, {d->w_dtype[0], d->w_dtype[1]}, 0, d->dim};
  hipStream_t st = (hipStream_t)stream;
  if (d->batch * d->seq) {
    for (int i = 0; i < 2; ++i) {
      if (int rc = check_tensor(who, i ? "k" : "q", d, d->x[i])) return rc;
      if (int rc = check_tensor(who, i ? "k's output's gradient" : "q's output's gradient", d, dy[i]))
        return rc;
    }
    SCAO_CHECK_ARG((!dw_q && !dw_k) || (workspace && (uintptr_t)workspace % 16 == 0),
                   "%s: workspace is null or not aligned", who);
    const int v = piece_of(*d);
    Args a = args_of(*d, BACKWARD_HEADS, v);
    for (int i = 0; i < 2; ++i) {
      to_out(a.s[i], dx[i]);
      to_dy(a.s[i], dy[i]);
    }
    j.blocks = backward_blocks(a);
    a.parts = dw_q || dw_k ? (float*)workspace : nullptr;
    j.parts = a.parts;
    for_variant(d->dtype, v, d->interleaved != 0, [&](auto type, auto piece, auto beside) {
      k_rope_backward<decltype(type)::value, decltype(piece)::value, decltype(beside)::value != 0>
          <<<j.blocks, THREADS, 0, st>>>(a);
    });
  }
  // (no token: the weights' gradients are zeros)
  if (dw_q || dw_k) k_rope_join<<<(2 * d->dim + 15) / 16, 16 * JOIN_ROWS, 0, st>>>(j);
  SCAO_LAUNCH_CHECK(who);
  return SCAO_OK;
}
