// The norm over all gradients of a model and their clipping to it, on gfx950.
//
//   N = scale * (sum over all tensors of sum |g|^p)^(1/p),  p = 1, 2, or the
//   largest |g|;  c = min(1, max_norm / (N + 1e-6));  g <- g * fp32(scale c)
//
// Two passes, because no element can be scaled before the last one is summed:
// k_norm reads every gradient and leaves one double per workgroup, k_scale
// adds those doubles (every workgroup all of them, in the same order: no
// atomics, no third launch) and reads and writes every gradient, or returns
// where the factor is exactly 1.  Both are bound by HBM.
//
// The tensors' table travels in the kernel's arguments, so a call copies
// nothing to the device and waits for nothing: at most TABLE tensors a launch.
// Each workgroup adds up for itself where a tensor's chunks begin, so that a
// tensor takes 12 bytes of it and not 20: 332 tensors of 25.5 MB in one table
// 25.5 us, in two tables of 190 40.2.  A tensor is cut into chunks of 32 KiB
// (eight 16-byte loads in flight a thread).  Vectors are aligned to 16 bytes
// whatever the tensor's start is: the first and the last vector of a tensor are
// taken element by element.
//
// Gradients that the last-level cache (256 MiB) holds: each workgroup takes a run
// of chunks, and the scaling begins with what was read last and writes through
// the caches.  Larger ones: the workgroups take chunks in turns, so that all of
// them read near each other, and the scaling goes past the caches, which would
// write the rest back while the next kernels read.  Gradients written, clipped
// and added to the parameters, runs through the caches against turns past them:
// 128 MB 196 us and 201, 200 MB 302 and 304, 268 MB 428 and 416, 400 MB 632 and
// 604; the clipping alone among others of its size, 268 MB 162 and 132 (6.1 TB/s
// for 3 x 268 MB).  Llama-1B's 2.47 GB in bf16: norm 419 us, 5.9 TB/s, both passes
// 1293, 5.7 TB/s; in runs through the caches 1453.
#include <algorithm>
#include <new>
#include <vector>

#include "../../include/scao_train.h"
#include "scao_common.hpp"

using namespace scao;

namespace {

constexpr int TABLE = 336;          // 12 bytes a tensor of the 4 KiB of arguments
constexpr int THREADS = 256;
constexpr int UNROLL = 8;
constexpr int CHUNK = THREADS * UNROLL;   // 16-byte vectors
constexpr int MAX_BLOCKS = 2048;    // eight workgroups a CU

struct Table {
  uint64_t ptr[TABLE];              // dtype in the two highest bits
  uint32_t numel[TABLE];            // larger tensors take several entries
  int32_t n, chunks, per;           // entries, chunks in all, chunks a run (0: in turns)
};
static_assert(sizeof(Table) <= 4096 - 40, "kernel arguments are limited to 4 KiB");
constexpr int64_t ENTRY = (int64_t)1 << 31;   // elements an entry

__host__ __device__ inline int size_of(int dt) { return dt == SCAO_F32 ? 4 : 2; }

// ------------------------------------------------------------ reduction ---
// p = 2: sum of squares in double (a square of two floats is exact there and
// cannot overflow or vanish); p = 1: sum of magnitudes in double; p = 0: the
// largest magnitude as its bit pattern, whose order is that of the values and
// in which a NaN is larger than infinity, so that it is not lost.
template <int P>
struct Acc {
  double s = 0.0;
  __device__ void add(float x) {
    if (P == 2) {
      const double d = (double)x;
      s = fma(d, d, s);
    } else {
      s += (double)fabsf(x);
    }
  }
  __device__ double value() const { return s; }
};
template <>
struct Acc<0> {
  uint32_t m = 0;
  __device__ void add(float x) { m = max(m, __float_as_uint(x) & 0x7fffffffu); }
  __device__ double value() const { return (double)m; }
};
template <int P>
__device__ __forceinline__ double join(double a, double b) {
  return P == 0 ? (a > b ? a : b) : a + b;
}
// of a workgroup, in an order of its own; every thread gets it
template <int P>
__device__ __forceinline__ double block_join(double x, double* lds) {
  for (int o = 32; o > 0; o >>= 1) x = join<P>(x, __shfl_xor(x, o, SCAO_WAVE));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  return join<P>(join<P>(join<P>(lds[0], lds[1]), lds[2]), lds[3]);
}
// N from the workgroups' parts
template <int P>
__device__ __forceinline__ double total_norm(const double* parts, int n, double scale,
                                             double* lds) {
  double x = 0.0;
  for (int i = threadIdx.x; i < n; i += THREADS) x = join<P>(x, parts[i]);
  x = block_join<P>(x, lds);
  if (P == 0) return (double)__uint_as_float((uint32_t)x) * scale;
  return (P == 2 ? sqrt(x) : x) * scale;
}

// ---------------------------------------------------------------- chunks ---
typedef __attribute__((address_space(1))) v4u_t gv4u;

template <int DT>
struct Values {
  static constexpr int E = DT == SCAO_F32 ? 4 : 8;
  static __device__ void get(v4u_t w, float (&x)[E]) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (DT == SCAO_F32) {
        x[t] = __uint_as_float(w[t]);
      } else if (DT == SCAO_BF16) {
        x[2 * t] = __uint_as_float(w[t] << 16);
        x[2 * t + 1] = __uint_as_float(w[t] & 0xffff0000u);
      } else {
        x[2 * t] = f16_to_f((uint16_t)w[t]);
        x[2 * t + 1] = f16_to_f((uint16_t)(w[t] >> 16));
      }
    }
  }
  static __device__ v4u_t put(const float (&x)[E]) {
    v4u_t w;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (DT == SCAO_F32)
        w[t] = __float_as_uint(x[t]);
      else if (DT == SCAO_BF16)
        w[t] = pk_bf16(x[2 * t], x[2 * t + 1]);
      else
        w[t] = (uint32_t)f_to_f16(x[2 * t]) | ((uint32_t)f_to_f16(x[2 * t + 1]) << 16);
    }
    return w;
  }
};

// One chunk of one tensor: f on every element, and with WRITE its result back
// in the element's place; PAST the caches or through them.
template <int DT, bool WRITE, bool PAST, class F>
__device__ __forceinline__ void each(uint64_t ptr, int64_t numel, int chunk, F&& f) {
  using V = Values<DT>;
  constexpr int E = V::E;
  const int64_t lo = (int64_t)(ptr & 15u) / (16 / E), hi = lo + numel;
  gv4u* base = (gv4u*)(ptr & ~(uint64_t)15);
  const int64_t v0 = (int64_t)chunk * CHUNK + threadIdx.x;
  const int64_t c0 = (int64_t)chunk * CHUNK * E;
  if (c0 >= lo && c0 + (int64_t)CHUNK * E <= hi) {
    v4u_t w[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      w[u] = PAST ? (v4u_t)__builtin_nontemporal_load(base + v0 + u * THREADS)
                  : (v4u_t)base[v0 + u * THREADS];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      float x[E];
      V::get(w[u], x);
#pragma unroll
      for (int t = 0; t < E; ++t) x[t] = f(x[t]);
      if (WRITE && PAST) __builtin_nontemporal_store(V::put(x), base + v0 + u * THREADS);
      else if (WRITE) base[v0 + u * THREADS] = V::put(x);
    }
    return;
  }
  for (int u = 0; u < UNROLL; ++u) {
    const int64_t v = v0 + u * THREADS, e = v * E;
    if (e >= hi) return;
    if (e >= lo && e + E <= hi) {
      float x[E];
      V::get(base[v], x);
#pragma unroll
      for (int t = 0; t < E; ++t) x[t] = f(x[t]);
      if (WRITE) base[v] = V::put(x);
    } else {
      for (int t = 0; t < E; ++t)
        if (e + t >= lo && e + t < hi) {
          const float y = f(ld1((void*)(ptr & ~(uint64_t)15), DT, e + t));
          if (WRITE) st1((void*)(ptr & ~(uint64_t)15), DT, e + t, y);
        }
    }
  }
}

__host__ __device__ inline int chunks_of(uint64_t ptr, int64_t numel, int dt) {
  static_assert(CHUNK * 16 == 1 << 15, "bytes of a chunk");
  const int bits = dt == SCAO_F32 ? 2 : 1;   // of an element's size
  const int64_t lo = (int64_t)(ptr & 15u) >> bits;
  return (int)((((lo + numel) << bits) + CHUNK * 16 - 1) >> 15);
}
// the chunks before each entry
__device__ __forceinline__ void count_chunks(const Table& tab, int* first) {
  static_assert(TABLE <= 2 * THREADS, "two entries a thread");
  __shared__ int waves[THREADS / 64];
  int own[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = 2 * threadIdx.x + i;
    own[i] = t < tab.n ? chunks_of(tab.ptr[t], tab.numel[t], (int)(tab.ptr[t] >> 62)) : 0;
  }
  int sum = own[0] + own[1];
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(sum, o, SCAO_WAVE);
    if ((int)(threadIdx.x & 63) >= o) sum += x;
  }
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 63) waves[wave] = sum;
  __syncthreads();
  int at = sum - own[0] - own[1];
  for (int w = 0; w < wave; ++w) at += waves[w];
  if (2 * (int)threadIdx.x < TABLE) first[2 * threadIdx.x] = at;
  if (2 * (int)threadIdx.x + 1 < TABLE) first[2 * threadIdx.x + 1] = at + own[0];
  __syncthreads();
}

// the workgroup's chunks, in the tensors that hold them
template <bool WRITE, bool PAST, class F>
__device__ __forceinline__ void walk(const Table& tab, int block, F&& f) {
  __shared__ int first[TABLE];
  count_chunks(tab, first);
  const int step = tab.per ? 1 : gridDim.x;
  int c = tab.per ? block * tab.per : block;
  const int end = tab.per ? min(c + tab.per, tab.chunks) : tab.chunks;
  int t = 0;
  for (int hi = tab.n; hi - t > 1;) {
    const int mid = (t + hi) >> 1;
    if (__builtin_amdgcn_readfirstlane(first[mid]) <= c) t = mid;
    else hi = mid;
  }
  for (; c < end; c += step) {
    while (t + 1 < tab.n && __builtin_amdgcn_readfirstlane(first[t + 1]) <= c) ++t;
    const int64_t numel = tab.numel[t];
    const uint64_t at = tab.ptr[t] & (~(uint64_t)0 >> 2);
    const int dt = (int)(tab.ptr[t] >> 62);
    const int chunk = c - __builtin_amdgcn_readfirstlane(first[t]);
    if (dt == SCAO_F32) each<SCAO_F32, WRITE, PAST>(at, numel, chunk, f);
    else if (dt == SCAO_BF16) each<SCAO_BF16, WRITE, PAST>(at, numel, chunk, f);
    else each<SCAO_F16, WRITE, PAST>(at, numel, chunk, f);
  }
}

template <int P>
__global__ __launch_bounds__(THREADS) void k_norm(const Table tab, double* parts) {
  __shared__ double lds[4];
  Acc<P> acc;
  walk<false, false>(tab, blockIdx.x, [&](float x) {
    acc.add(x);
    return x;
  });
  const double x = block_join<P>(acc.value(), lds);
  if (threadIdx.x == 0) parts[blockIdx.x] = x;
}

template <int P>
__global__ __launch_bounds__(THREADS) void k_norm_out(const double* parts, int nparts,
                                                      double scale, float* norm) {
  __shared__ double lds[4];
  const double n = total_norm<P>(parts, nparts, scale, lds);
  if (threadIdx.x == 0) *norm = (float)n;
}

template <int P, bool PAST>
__global__ __launch_bounds__(THREADS) void k_scale(const Table tab, const double* parts,
                                                   int nparts, double scale, double max_norm,
                                                   float* norm) {
  __shared__ double lds[4];
  const double n = total_norm<P>(parts, nparts, scale, lds);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  // (max_norm infinite: the factor is scale, with an infinite norm too)
  const double c = max_norm / (n + 1e-6);
  const float factor = (float)(c < 1.0 || n != n ? scale * c : scale);
  if (factor == 1.0f) return;
  walk<true, PAST>(tab, gridDim.x - 1 - blockIdx.x, [&](float x) { return x * factor; });
}

// ------------------------------------------------------------------ host ---
int chunks_of(const scao_tensor_desc& t) {
  int64_t n = 0;
  for (int64_t at = 0; at < t.numel; at += ENTRY)
    n += chunks_of((uint64_t)(uintptr_t)t.data, std::min(ENTRY, t.numel - at), t.dtype);
  return (int)n;
}

int check(const char* who, const scao_tensor_desc* t, int n, int norm_type, double scale) {
  SCAO_CHECK_ARG(n >= 0 && (n == 0 || t), "%s: null table or negative count", who);
  SCAO_CHECK_ARG(norm_type >= 0 && norm_type <= 2, "%s: norm type %d is not 0, 1 or 2",
                 who, norm_type);
  SCAO_CHECK_ARG(scale > 0.0 && scale <= 1.7e308, "%s: scale %g is not positive and finite",
                 who, scale);
  int64_t chunks = 0;
  for (int i = 0; i < n; ++i) {
    SCAO_CHECK_ARG(t[i].dtype >= 0 && t[i].dtype <= SCAO_F16, "%s: dtype %d of tensor %d", who,
                   t[i].dtype, i);
    SCAO_CHECK_ARG(t[i].numel >= 0 && t[i].numel < ((int64_t)1 << 40),
                   "%s: size of tensor %d", who, i);
    if (t[i].numel == 0) continue;
    SCAO_CHECK_ARG(t[i].data && (uintptr_t)t[i].data % size_of(t[i].dtype) == 0,
                   "%s: tensor %d is null or not aligned to its elements", who, i);
    SCAO_CHECK_ARG((uint64_t)(uintptr_t)t[i].data >> 57 == 0, "%s: address of tensor %d", who, i);
    chunks += chunks_of(t[i]);
  }
  SCAO_CHECK_ARG(chunks < ((int64_t)1 << 30), "%s: more than 32 TiB of gradients", who);
  return SCAO_OK;
}

int check_buffers(const char* who, int n, const float* norm, const void* workspace) {
  SCAO_CHECK_ARG(norm && (workspace || n == 0), "%s: null pointer", who);
  SCAO_CHECK_ARG((uintptr_t)norm % 4 == 0 && (uintptr_t)workspace % 8 == 0,
                 "%s: norm or workspace is not aligned", who);
  return SCAO_OK;
}

// No element may be scaled twice, nor by two workgroups at once.  Tensors in the
// order of their addresses, or against it, as a backward pass often allocates
// them, need no sorting (332 tensors: 16 us).
int check_apart(const scao_tensor_desc* t, int n) try {
  auto begin = [&](int i) { return (uintptr_t)t[i].data; };
  auto end = [&](int i) { return (uintptr_t)t[i].data + t[i].numel * size_of(t[i].dtype); };
  bool up = true, down = true;
  for (int i = 0, last = -1; i < n; ++i) {
    if (!t[i].numel) continue;
    if (last >= 0) {
      up = up && begin(i) >= end(last);
      down = down && begin(last) >= end(i);
    }
    last = i;
  }
  if (up || down) return SCAO_OK;
  std::vector<std::pair<uintptr_t, uintptr_t>> r;
  r.reserve(n);
  for (int i = 0; i < n; ++i)
    if (t[i].numel) r.emplace_back(begin(i), end(i));
  std::sort(r.begin(), r.end());
  for (size_t i = 1; i < r.size(); ++i)
    SCAO_CHECK_ARG(r[i].first >= r[i - 1].second, "scao_grad_clip: two gradients share memory");
  return SCAO_OK;
} catch (const std::bad_alloc&) {
  scao_set_error("scao_grad_clip: no host memory for %d tensors", n);
  return SCAO_ERR_INVALID;
}

// more than the last-level cache can keep beside what else a step moves
bool large(const scao_tensor_desc* t, int n) {
  int64_t bytes = 0;
  for (int i = 0; i < n; ++i) bytes += t[i].numel * size_of(t[i].dtype);
  return bytes > ((int64_t)192 << 20);
}

template <class F>
int for_launches(const scao_tensor_desc* t, int n, F&& f) {
  const bool turns = large(t, n);
  Table tab;
  int i = 0;
  int64_t at = 0;   // of tensor i
  while (i < n) {
    tab.n = tab.chunks = 0;
    while (i < n && tab.n < TABLE) {
      const int64_t m = std::min(ENTRY, t[i].numel - at);
      if (m > 0) {
        const uint64_t p = (uint64_t)(uintptr_t)t[i].data + at * size_of(t[i].dtype);
        tab.ptr[tab.n] = p | (uint64_t)t[i].dtype << 62;
        tab.numel[tab.n++] = (uint32_t)m;
        tab.chunks += chunks_of(p, m, t[i].dtype);
        at += m;
      }
      if (at >= t[i].numel) {
        ++i;
        at = 0;
      }
    }
    if (!tab.n) break;
    const int per = (tab.chunks + MAX_BLOCKS - 1) / MAX_BLOCKS;
    tab.per = turns ? 0 : per;
    const int rc = f(tab, (tab.chunks + per - 1) / per);
    if (rc) return rc;
  }
  return SCAO_OK;
}

int norm_parts(const scao_tensor_desc* t, int n, int norm_type, double* parts, int* nparts,
               hipStream_t st) {
  *nparts = 0;
  return for_launches(t, n, [&](const Table& tab, int blocks) -> int {
    double* out = parts + *nparts;
    if (norm_type == 2) k_norm<2><<<blocks, THREADS, 0, st>>>(tab, out);
    else if (norm_type == 1) k_norm<1><<<blocks, THREADS, 0, st>>>(tab, out);
    else k_norm<0><<<blocks, THREADS, 0, st>>>(tab, out);
    SCAO_LAUNCH_CHECK("scao_grad_norm");
    *nparts += blocks;
    return SCAO_OK;
  });
}

}  // namespace

extern "C" int64_t scao_grad_norm_workspace(const scao_tensor_desc* tensors, int n) {
  if (n <= 0 || !tensors) return 0;
  int64_t entries = 1;   // a call with empty tensors alone has a workspace too
  for (int i = 0; i < n; ++i)
    if (tensors[i].numel > 0) entries += (tensors[i].numel - 1) / ENTRY + 1;
  if (entries > 1) --entries;
  // every launch leaves at most MAX_BLOCKS doubles
  return (entries + TABLE - 1) / TABLE * MAX_BLOCKS * (int64_t)sizeof(double);
}

extern "C" int scao_grad_norm(const scao_tensor_desc* tensors, int n, int norm_type, double scale,
                              float* norm, void* workspace, void* stream) {
  if (int rc = check("scao_grad_norm", tensors, n, norm_type, scale)) return rc;
  if (int rc = check_buffers("scao_grad_norm", n, norm, workspace)) return rc;
  hipStream_t st = (hipStream_t)stream;
  double* parts = (double*)workspace;
  int np = 0;
  if (int rc = norm_parts(tensors, n, norm_type, parts, &np, st)) return rc;
  if (norm_type == 2) k_norm_out<2><<<1, THREADS, 0, st>>>(parts, np, scale, norm);
  else if (norm_type == 1) k_norm_out<1><<<1, THREADS, 0, st>>>(parts, np, scale, norm);
  else k_norm_out<0><<<1, THREADS, 0, st>>>(parts, np, scale, norm);
  SCAO_LAUNCH_CHECK("scao_grad_norm");
  return SCAO_OK;
}

extern "C" int scao_grad_clip(const scao_tensor_desc* tensors, int n, int norm_type, double scale,
                              double max_norm, float* norm, void* workspace, void* stream) {
  if (int rc = check("scao_grad_clip", tensors, n, norm_type, scale)) return rc;
  SCAO_CHECK_ARG(max_norm >= 0.0, "scao_grad_clip: max_norm %g is negative or no number", max_norm);
  if (int rc = check_buffers("scao_grad_clip", n, norm, workspace)) return rc;
  if (int rc = check_apart(tensors, n)) return rc;
  hipStream_t st = (hipStream_t)stream;
  double* parts = (double*)workspace;
  int np = 0;
  if (int rc = norm_parts(tensors, n, norm_type, parts, &np, st)) return rc;
  if (np == 0) return scao_grad_norm(tensors, 0, norm_type, scale, norm, nullptr, stream);
  float* out = norm;
  const bool past = large(tensors, n);
  return for_launches(tensors, n, [&](const Table& tab, int blocks) -> int {
#define SCALE(P)                                                                              \
  past ? k_scale<P, true><<<blocks, THREADS, 0, st>>>(tab, parts, np, scale, max_norm, out)   \
       : k_scale<P, false><<<blocks, THREADS, 0, st>>>(tab, parts, np, scale, max_norm, out)
    if (norm_type == 2) SCALE(2);
    else if (norm_type == 1) SCALE(1);
    else SCALE(0);
#undef SCALE
    SCAO_LAUNCH_CHECK("scao_grad_clip");
    out = nullptr;   // the first launch's first workgroup writes it
    return SCAO_OK;
  });
}
