// Times of the orthogonalisation's products on either tile in every number of parts, and of
// its steps by panels: what the constants of csrc/ortho.hip's choice were fitted to.  One
// CSV row a form on stdout, the least of three runs.  A list is (rows x cols * how many)s
// of one or two words an element.
//
//   hipcc --offload-arch=gfx950 -O3 -std=c++17 -ffp-contract=off -Xclang
//     -target-feature -Xclang -packed-fp32-ops -o ortho_tiles perf/ortho_tiles.hip
#include <stdio.h>
#include <stdlib.h>

#include "../scao_amd/csrc/ortho.hip"
#include "../scao_amd/csrc/ortho_tiles128.hip"
#include "../scao_amd/csrc/ortho_tiles256.hip"

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

const char* LISTS[] = {
    "256x256*1", "256x256*16", "256x256*64", "160x160*1", "160x160*16", "144x1024*8", "300x700*2",
    "384x384*1", "384x384*8", "512x512*1", "512x512*4", "512x512*40", "512x256*8", "256x1024*4",
    "512x1024*4", "320x640*8", "640x640*1", "640x640*30", "1024x1024*1", "1024x1024*4",
    "1024x1024*8", "1024x1024*16", "1024x1024*20", "512x2048*8", "2048x2048*1", "2048x2048*2",
    "2048x2048*4", "2048x2048*8", "336x1000*12", "1001x333*12,333x1001*5,77x2049*7",
    "768x2304*12,768x768*12", "6246x384*4,599x256*16", "384x1536*4,448x1024*4,1593x2112*1",
    "63x1599*16,320x46*3", "1024x4096*4", "2048x8192*4", "14336x4096*1"};

constexpr int64_t ROOM = (int64_t)4 << 30, PARTS = (int64_t)512 << 20;
char *buffer, *parts_buffer;

// fp16 numbers, uniform in -1 .. 1
__global__ void fill(uint16_t* p, int64_t n) {
  const int64_t i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= n) return;
  uint32_t x = (uint32_t)i * 2654435761u;
  x ^= x >> 16;
  x *= 0x85ebca6bu;
  x ^= x >> 13;
  x *= 0xc2b2ae35u;
  x ^= x >> 16;
  p[i] = f_to_f16((float)(x >> 8) * (2.f / 16777216.f) - 1.f);
}

std::vector<Matrix> matrices_of(const char* list, int words) {
  std::vector<Matrix> m;
  for (const char* at = list; *at;) {
    char* end;
    const int64_t rows = strtol(at, &end, 10), cols = strtol(end + 1, &end, 10);
    const int many = (int)strtol(end + 1, &end, 10);
    const int w = words_of(words == 2 ? SCAO_ORTHO_FP32 : SCAO_ORTHO_FAST, rows, cols);
    for (int i = 0; i < many; ++i)
      m.push_back({nullptr, nullptr, nullptr, rows, cols, cols, cols, SCAO_F32, SCAO_F32, 0.f, 0.f, w});
    at = *end ? end + 1 : end;
  }
  return m;
}

template <class F>
float time_of(F&& run) {
  hipEvent_t begin, end;
  CHECK(hipEventCreate(&begin));
  CHECK(hipEventCreate(&end));
  run();
  run();
  float best = 1e9f;
  for (int r = 0; r < 3; ++r) {
    CHECK(hipEventRecord(begin));
    for (int i = 0; i < 6; ++i) run();
    CHECK(hipEventRecord(end));
    CHECK(hipEventSynchronize(end));
    float ms;
    CHECK(hipEventElapsedTime(&ms, begin, end));
    best = std::min(best, ms * 1e3f / 6);
  }
  CHECK(hipGetLastError());
  CHECK(hipEventDestroy(begin));
  CHECK(hipEventDestroy(end));
  return best;
}

void sweep(const char* list, int words) {
  const std::vector<Matrix> m = matrices_of(list, words);
  const OrthoOut out{};
  for_passes(m, [&](const int* order, int n) -> int {
    if (n != (int)m.size()) {
      fprintf(stderr, "%s: more than a pass\n", list);
      exit(1);
    }
    Pass p(m.data(), order, n, buffer, true);
    Plan never[3];
    for (Plan& q : never) q.us = 1e30;
    const std::vector<PanelGroup> panels = p.panels_of(never);
    if (p.peak > ROOM) {
      fprintf(stderr, "%s: too large\n", list);
      exit(1);
    }
    for (int phase = 0; phase < 3; ++phase)
      for (int big = 0; big < 2; ++big) {
        const int side = COSTS[0][big].side, slots = COSTS[0][big].slots;
        OrthoPhase ph{};
        p.lay(phase, side, ph);
        ph.base = buffer;
        ph.partial = (float*)parts_buffer;
        // results stay in -1 .. 1
        int k = 0;
        for (const OrthoGroup& g : p.groups)
          k = std::max(k, phase == ORTHO_GRAM ? std::max(g.rows, g.cols) : std::min(g.rows, g.cols));
        ph.by = 1.f / k;
        for (int parts : {1, 2, 3, 4, 6, 8, 12, 16})
          for (int whole : {0, ph.tiles / slots * slots}) {
            if (parts == 1 ? whole != 0 : whole == ph.tiles) continue;
            const int64_t rest = ph.tiles - whole;
            if (parts > 1 && (rest * parts > (big ? 1024 : 2048) ||
                              2 * parts > Pass::steps_of(phase, ph.g[0]) ||
                              rest * parts * side * side * 4 > PARTS))
              continue;
            OrthoPhase q = ph;
            q.splits = parts;
            q.whole = parts == 1 ? ph.tiles : whole;
            const float us = time_of(
                [&] { (big ? ortho_tiles256 : ortho_tiles128)(phase, ORTHO_NEXT, q, out, 0); });
            printf("\"%s\",%d,%d,%d,%d,%d,%.1f\n", list, words, phase, side, parts,
                   parts == 1 ? ph.tiles : whole, us);
            if (ph.tiles < slots) break;   // (the same again)
          }
      }
    // a whole step by panels, if they can hold these matrices
    if (panels.empty()) return SCAO_OK;
    OrthoPanels a{};
    int blocks = 0, lds = 0;
    bool all = true;
    for (const PanelGroup& q : panels) {
      all = all && panel_held(q);
      a.g[a.groups++] = q;
      blocks += q.per * q.count;
      lds = std::max(lds, panel_lds(q));
    }
    a.base = buffer;
    a.gram = 1.f / 1024;
    a.second = a.third = 1.f / 512;
    a.a = 1.f;
    auto* kernel = all ? k_ortho_panels<true, ORTHO_NEXT> : k_ortho_panels<false, ORTHO_NEXT>;
    printf("\"%s\",%d,panels,16,1,0,%.1f\n", list, words,
           time_of([&] { kernel<<<blocks, PANEL_THREADS, lds, 0>>>(a, out); }));
    return SCAO_OK;
  });
  fflush(stdout);
}

}  // namespace

int main() {
  CHECK(hipMalloc(&buffer, ROOM));
  CHECK(hipMalloc(&parts_buffer, PARTS));
  fill<<<(int)(ROOM / 2 / 256), 256>>>((uint16_t*)buffer, ROOM / 2);
  CHECK(hipDeviceSynchronize());
  printf("list,words,phase,side,parts,whole,us\n");
  for (const char* list : LISTS)
    for (int words : {1, 2}) sweep(list, words);
}
