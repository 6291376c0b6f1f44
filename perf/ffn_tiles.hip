// Times of the feed-forward block's products on every tile in every number of
// parts, bf16: what the constants of csrc/ffn.hip's choice were fitted to. One CSV
// row a form on stdout. 45 blocks of 8 to 4096 tokens and five shapes; the least
// of three runs, weights taken from four copies in turn.
//
//   hipcc --offload-arch=gfx950 -O3 -std=c++17 -ffp-contract=off -Xclang
//     -target-feature -Xclang -packed-fp32-ops -o ffn_tiles perf/ffn_tiles.hip
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
#include <vector>

#include "../scao_amd/csrc/ffn_kernels.hpp"

using namespace scao;

void scao_set_error(const char*, ...) {}

#define CHECK(x)                                                                       \
  do {                                                                                 \
    const hipError_t e_ = (x);                                                         \
    if (e_ != hipSuccess) {                                                            \
      fprintf(stderr, "line %d: %s\n", __LINE__, hipGetErrorString(e_));               \
      exit(1);                                                                         \
    }                                                                                  \
  } while (0)

namespace {

const char* KINDS[] = {"gate_up", "down", "dh", "dx", "dw"};
const char* TILES[FFN_TILES] = {"256x256", "256x128", "128x128", "64x128", "32x128"};

// uniform in -1 .. 1
__global__ void fill(uint16_t* p, int64_t n) {
  const int64_t i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= n) return;
  uint32_t x = (uint32_t)i * 2654435761u;
  x ^= x >> 16;
  x *= 0x85ebca6bu;
  x ^= x >> 13;
  x *= 0xc2b2ae35u;
  x ^= x >> 16;
  p[i] = f_to_bf16((float)(x >> 8) * (2.f / 16777216.f) - 1.f);
}

constexpr int64_t ROOM = (int64_t)6 << 30, PARTS = (int64_t)1 << 30;
char* buffer;

void sweep(int kind, int tokens, int d, int f) {
  const bool gated = kind == FFN_GATE_UP, over_f = kind == FFN_DOWN || kind == FFN_DX;
  FfnOperands o{};
  FfnEpilogue e{};
  o.M = kind == FFN_DW ? 2 * f : tokens;
  o.N = kind == FFN_GATE_UP || kind == FFN_DH ? f : d;
  o.K = kind == FFN_DW ? tokens : over_f ? f : d;
  o.nseg = kind == FFN_DX ? 2 : 1;
  int64_t used = 0;
  auto take = [&](int64_t bytes) {
    char* p = buffer + used;
    used += (bytes + 255) / 256 * 256;
    if (used > ROOM) {
      fprintf(stderr, "too large\n");
      exit(1);
    }
    return p;
  };
  const int64_t weights = (int64_t)o.N * o.K * 2;
  char* a = take((int64_t)o.M * o.K * 2 * o.nseg);
  e.out = take((int64_t)o.M * o.N * 2 * (kind == FFN_DH ? 2 : 1));
  e.ldo = kind == FFN_DH ? 2 * o.N : o.N;
  e.rows = o.M;
  e.second = 0x7fffffff;
  e.cols = o.N;
  if (kind == FFN_DH) {
    e.fi = (tokens + 15) / 16;
    e.fj = (f + 15) / 16;
    e.ab = take(ab_bytes<SCAO_BF16>(e.fi, e.fj));
  }
  e.partial = (float*)take(PARTS);
  o.lda = kind == FFN_DX ? 2 * f : kind == FFN_DW ? o.M : o.K;
  o.ldb = kind == FFN_GATE_UP || kind == FFN_DOWN ? o.K : o.N;
  std::vector<FfnOperands> copies(4, o);
  for (FfnOperands& c : copies) {
    char* w = take(weights * (gated || kind == FFN_DX ? 2 : 1));
    c.a[0] = a;
    c.b[0] = w;
    c.a[1] = a + f * 2;
    c.b[1] = w + weights;
    c.b[FFN_MAX_SEG / 2] = w + weights;
  }

  const int steps = o.nseg * ((o.K + FFN_BK - 1) / FFN_BK);
  const double gflop = 2.0 * o.M * o.N * o.K * o.nseg * (gated ? 2 : 1) / 1e9;
  const int reps = gflop > 500 ? 4 : 8;
  hipEvent_t begin, end;
  CHECK(hipEventCreate(&begin));
  CHECK(hipEventCreate(&end));
  for (int tile = 0; tile < FFN_TILES; ++tile) {
    // (launch_tile has no others)
    if (kind == FFN_DW && tile != FFN_256x256 && tile != FFN_128x128) continue;
    if (tile == FFN_256x128 && kind != FFN_DOWN) continue;
    if (FFN_BM[tile] > 32 && 4 * o.M <= FFN_BM[tile]) continue;
    const int cols = gated ? FFN_BN[tile] / 2 : FFN_BN[tile];
    const int tm = (o.M + FFN_BM[tile] - 1) / FFN_BM[tile], tn = (o.N + cols - 1) / cols;
    for (int parts : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
      if (parts > 1 && (parts * 2 > steps || tm * tn * parts > 2048)) break;
      if (parts > 1 && (int64_t)parts * tm * tn * FFN_BM[tile] * FFN_BN[tile] * 4 > PARTS) break;
      auto run = [&](int c) {
        FfnOperands q = copies[c % copies.size()];
        q.tiles_m = tm;
        q.tiles_n = tn;
        q.splits = parts;
        q.whole = parts == 1 ? tm * tn : 0;
        launch_product<SCAO_BF16>(kind, tile, q, e, 0);
      };
      run(0);
      run(1);
      CHECK(hipDeviceSynchronize());
      float best = 1e9f;
      for (int r = 0; r < 3; ++r) {
        CHECK(hipEventRecord(begin));
        for (int c = 0; c < reps; ++c) run(c);
        CHECK(hipEventRecord(end));
        CHECK(hipEventSynchronize(end));
        float ms;
        CHECK(hipEventElapsedTime(&ms, begin, end));
        best = std::min(best, ms * 1e3f / reps);
      }
      printf("%s,%d,%d,%d,%s,%d,%.1f\n", KINDS[kind], tokens, d, f, TILES[tile], parts, best);
    }
  }
  fflush(stdout);
  CHECK(hipEventDestroy(begin));
  CHECK(hipEventDestroy(end));
}

}  // namespace

int main() {
  CHECK(hipMalloc(&buffer, ROOM));
  fill<<<(int)(ROOM / 2 / 256), 256>>>((uint16_t*)buffer, ROOM / 2);
  CHECK(hipDeviceSynchronize());
  printf("product,tokens,d,f,tile,parts,us\n");
  const int shapes[][2] = {{2048, 8192}, {4096, 14336}, {1024, 2816}, {768, 2048}, {256, 704}};
  for (const auto& s : shapes)
    for (int tokens : {8, 24, 64, 128, 256, 512, 1024, 2048, 4096})
      for (int kind = 0; kind < 5; ++kind) sweep(kind, tokens, s[0], s[1]);
}
