// Newton-Schulz orthogonalisation of matrix updates, and the step of the optimiser
// that is built on it: argument checks, memory plans and the order of the launches.
// The kernels are in ortho_kernels.hpp, ortho_norm.hpp, ortho_small.hpp and
// ortho_panels.hpp.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "ortho_panels.hpp"

using namespace scao;

namespace {

constexpr int MAX_STEPS = 64;
constexpr int64_t MAX_SIDE = (int64_t)1 << 20, MAX_SMALLER = (int64_t)1 << 15;

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
int size_of(int dt) { return dt == SCAO_F32 ? 4 : 2; }

struct Matrix {
  const void* src;
  float* buf;
  void* dst;
  int64_t rows, cols, ld_src, ld_dst;
  int src_dtype, dst_dtype;
  float rate, decay;
  int words;
  int64_t smaller() const { return std::min(rows, cols); }
  int64_t larger() const { return std::max(rows, cols); }
  // C's tiles of 256 x 256 in an update
  int64_t tiles() const { return ((rows + 255) / 256) * ((cols + 255) / 256); }
};

// ------------------------------------------------- what the words can hold ---
// The largest |f| on [0, u] of an odd polynomial a x + b x^3 + c x^5.
double largest(double a, double b, double c, double u) {
  auto at = [&](double x) { return std::fabs(x * (a + x * x * (b + x * x * c))); };
  double most = at(u);
  // a + 3 b t + 5 c t^2 = 0, t = x^2
  double t[2] = {-1, -1};
  const double p = 5 * c, q = 3 * b, disc = q * q - 4 * p * a;
  if (p == 0) {
    if (q != 0) t[0] = -a / q;
  } else if (disc >= 0) {
    const double z = -0.5 * (q + std::copysign(std::sqrt(disc), q));
    t[0] = z / p;
    if (z != 0) t[1] = a / z;
  }
  for (double x : t)
    if (x > 0 && x < u * u) most = std::max(most, at(std::sqrt(x)));
  return most;
}
// of a + b t + c t^2 on [0, t0]
double largest2(double a, double b, double c, double t0) {
  auto at = [&](double t) { return std::fabs(a + t * (b + t * c)); };
  double most = std::max(at(0), at(t0));
  if (c != 0) {
    const double t = -b / (2 * c);
    if (t > 0 && t < t0) most = std::max(most, at(t));
  }
  return most;
}
// a power of two that takes values up to `most` to at most 16384, a quarter of
// fp16's range: what the roundings before it have added finds room
double power_for(double most, int limit) {
  if (!(most > 0)) return std::ldexp(1.0, limit);
  return std::ldexp(1.0, std::min(limit, (int)std::floor(std::log2(16384.0 / most))));
}
struct Scales {
  double first;                       // of the first X
  float gram[MAX_STEPS], square[MAX_STEPS], square_keep[MAX_STEPS];
  float diagonal[MAX_STEPS], update[MAX_STEPS];
  // by panels: of A X and (A X) X^T as words; of X, A X and A A X in the next X
  float second[MAX_STEPS], third[MAX_STEPS], a[MAX_STEPS], b[MAX_STEPS], c[MAX_STEPS];
};
// false: some singular value may grow past what the words hold
bool scales_of(const double* co, int steps, Scales& s) {
  double u = 1.0, sx = power_for(u, 14);
  s.first = sx;
  for (int k = 0; k < steps; ++k) {
    const double a = co[3 * k], b = co[3 * k + 1], c = co[3 * k + 2];
    const double sa = power_for(u * u, 14), sb = power_for(largest2(a, b, c, u * u), 20);
    const double next = largest(a, b, c, u) * 1.01;
    if (!(next <= 1024.0) || !(sb >= 1.0 / 65536)) return false;
    const double to = k + 1 < steps ? power_for(next, 14) : 1.0;
    s.gram[k] = (float)(sa / (sx * sx));
    s.square[k] = (float)(c * sb / (sa * sa));
    s.square_keep[k] = (float)(b * sb / sa);
    s.diagonal[k] = (float)(a * sb);
    s.update[k] = (float)(to / (sb * sx));
    const double sy = power_for(u * u * u, 28), sz = power_for(u * u * u * u, 28);
    s.second[k] = (float)(sy / (sa * sx));
    s.third[k] = (float)(sz / (sy * sx));
    s.a[k] = (float)(a * to / sx);
    s.b[k] = (float)(b * to / (sa * sx));
    s.c[k] = (float)(c * to / (sz * sx));
    u = next;
    sx = to;
  }
  return true;
}

// -------------------------------------------------------------- one pass ---
// Estimated us of the products' tiles, by words and tile: of a k step (64 k, or 32 of
// two words) with a CU's LDS to one tile and with all it holds, and of a tile's beginning
// and end (sums alone, an update's, a symmetric product's with its image); of a join, a
// part and element.  Fitted to launches of 10 to 1296 tiles and 6 to 72 steps; of the 222
// launches of profiles/ortho_tiles.csv (perf/ortho_tiles.hip measured them) the chosen
// form is 0.8% behind the best one on the geometric average, 18% at most.
struct Cost {
  int side, slots;
  double lone, full, parts, update, symmetric;
  // 128 x 128 tiles: two on a CU as soon as there are more than CUs
  double step(int64_t groups) const {
    if (slots > 256) return groups > 256 ? full : lone;
    return lone + (full - lone) * std::min(1.0, groups / 256.0);
  }
};
const Cost COSTS[2][2] = {{{128, 512, 0.50, 0.94, 6.5, 6.5, 7.5}, {256, 256, 1.00, 1.40, 13, 13, 16}},
                          {{128, 512, 0.67, 1.28, 6.5, 8.0, 9.0}, {256, 256, 1.60, 2.18, 13, 16, 24}}};
const double JOIN[2] = {0.87e-6, 1.6e-6};
// k steps of two words that a 256 x 256 tile adds up in the matrix cores, whose errors
// grow with the root of a sum's length: such a tile has no registers to put sums aside
// (128 x 128 tiles do, every eight steps).  The published
// five steps in fp32: with Gram matrices on 256 x 256 tiles results of 512 x 2048 (64
// steps) are 2.2e-6 off where 128 x 128 tiles leave 1.7e-6, of 512 x 14336 (448) 5.7e-6
// and 1.7e-6, of 512 x 65536 1.1e-5 and 2.1e-6; all phases on 256 x 256 tiles, 2048 x 2048
// (64) 2.4e-6 and 0.9e-6, 4096 x 4096 (128) 3.3e-6 and 1.0e-6 (in a library's products
// 3.6e-6 and 4.8e-6).  Longer sums take smaller tiles, or parts, which are joined with
// rounding: two of 4096 x 4096 take a sixth longer so, two of 4096 x 14336 a quarter.
constexpr int64_t LONG_SUM = 64;

struct Plan {
  int big = 0;
  double us = 0;
  OrthoPhase ph{};
};

bool same_group(const Matrix& a, const Matrix& b) {
  return a.rows == b.rows && a.cols == b.cols && a.words == b.words;
}

struct Pass {
  const Matrix* m;
  const int* order;          // the pass's entries
  int n;
  char* base;
  std::vector<OrthoGroup> groups;
  double* norms = nullptr;
  int64_t used = 0, peak = 0;

  int64_t take(int64_t bytes) {
    const int64_t at = used;
    used += round_up(bytes, 256);
    peak = std::max(peak, used);
    return at;
  }
  const Matrix& entry(int i) const { return m[order[i]]; }

  Pass(const Matrix* matrices, const int* order_, int n_, char* base_, bool again)
      : m(matrices), order(order_), n(n_), base(base_) {
    norms = (double*)(base + take((int64_t)ORTHO_MATRICES * ORTHO_PARTS * 8));
    for (int i = 0; i < n;) {
      OrthoGroup g{};
      g.first = i;
      g.rows = (int)entry(i).rows;
      g.cols = (int)entry(i).cols;
      g.words = entry(i).words;
      while (i < n && same_group(entry(i), entry(g.first))) ++i;
      g.count = i - g.first;
      const int64_t s = std::min(g.rows, g.cols);
      g.ldx = (int)round_up(g.cols, 8);
      g.lda = (int)round_up(s, 8);
      g.x_step = round_up((int64_t)g.words * g.rows * g.ldx * 2, 256);
      g.a_step = round_up(g.words * s * g.lda * 2, 256);
      g.x = take(g.count * g.x_step);
      g.y = again ? take(g.count * g.x_step) : g.x;   // (one step writes the result alone)
      g.a = take(g.count * g.a_step);
      g.b = take(g.count * g.a_step);
      groups.push_back(g);
    }
  }

  // k steps of a tile
  static int64_t steps_of(int phase, const OrthoGroup& g) {
    const int k = phase == ORTHO_GRAM ? std::max(g.rows, g.cols) : std::min(g.rows, g.cols);
    const int bk = FFN_BK / g.words;
    return (k + bk - 1) / bk;
  }
  // The groups' tiles of `side`, the longest sums first.
  void lay(int phase, int side, OrthoPhase& ph) const {
    std::vector<OrthoGroup> g = groups;
    std::stable_sort(g.begin(), g.end(), [&](const OrthoGroup& a, const OrthoGroup& b) {
      return steps_of(phase, a) > steps_of(phase, b);
    });
    int64_t tiles = 0;
    for (size_t i = 0; i < g.size(); ++i) {
      OrthoGroup& q = g[i];
      if (phase == ORTHO_UPDATE) {
        q.tiles_m = (q.rows + side - 1) / side;
        q.tiles_n = (q.cols + side - 1) / side;
        q.per = q.tiles_m * q.tiles_n;
      } else {
        q.tiles_m = q.tiles_n = (int)((std::min(q.rows, q.cols) + side - 1) / side);
        q.per = q.tiles_m * (q.tiles_m + 1) / 2;
      }
      q.tile0 = (int)tiles;
      tiles += (int64_t)q.count * q.per;
      ph.g[i] = q;
    }
    ph.groups = (int)g.size();
    ph.tiles = (int)tiles;
  }
  // Estimated us of the tiles from `begin` on, each in n parts: rounds of as many
  // workgroups as the chip holds, as long as their first, with the CUs shared by as many
  // as would do the round's steps at that length (a few long tiles among short ones have
  // their CUs alone: 4 Gram matrices of 384 over 6246 rows and 16 of 256 over 599).
  static double rounds(int phase, const OrthoPhase& ph, int big, int begin, int end, int n) {
    double us = 0;
    int k = 0;
    const int64_t slots = COSTS[0][big].slots, stop = (int64_t)end * n;
    for (int64_t at = (int64_t)begin * n; at < stop; at += slots) {
      while (k + 1 < ph.groups && (int64_t)ph.g[k + 1].tile0 * n <= at) ++k;
      const int64_t last = std::min(stop, at + slots);
      const Cost& c = COSTS[ph.g[k].words - 1][big];
      const int first = (steps_of(phase, ph.g[k]) + n - 1) / n;
      int64_t steps = 0;
      for (int i = k; i < ph.groups && (int64_t)ph.g[i].tile0 * n < last; ++i) {
        const int64_t from = std::max(at, (int64_t)ph.g[i].tile0 * n);
        const int64_t to = i + 1 < ph.groups ? std::min(last, (int64_t)ph.g[i + 1].tile0 * n) : last;
        steps += (to - from) * ((steps_of(phase, ph.g[i]) + n - 1) / n);
      }
      us += first * c.step(steps / first) +
            (n > 1 ? c.parts : phase == ORTHO_UPDATE ? c.update : c.symmetric);
    }
    return us;
  }
  // Which tile, how many of them run in one piece and in how many parts the others:
  // all of them, or those that do not fill a last round.
  Plan plan(int phase) {
    Plan best;
    double least = 1e30;
    for (int big = 0; big < 2; ++big) {
      const int side = COSTS[0][big].side, slots = COSTS[0][big].slots;
      OrthoPhase ph{};
      lay(phase, side, ph);
      int64_t sum = 0;   // the longest of two words
      for (const OrthoGroup& g : groups)
        if (g.words == 2) sum = std::max(sum, steps_of(phase, g));
      const int whole_rounds = ph.tiles / slots * slots;
      for (int n : {1, 2, 3, 4, 6, 8, 12, 16})
        for (int whole : {0, whole_rounds}) {
          if (n == 1 ? whole != 0 : whole == ph.tiles) continue;
          if (big && (whole || n == 1 ? sum : (sum + n - 1) / n) > LONG_SUM) continue;
          const int rest = ph.tiles - whole;
          if (n > 1 && ((int64_t)rest * n > (big ? 1024 : 2048) ||
                        2 * n > steps_of(phase, ph.g[0])))
            continue;
          double us = n == 1 ? rounds(phase, ph, big, 0, ph.tiles, 1)
                             : rounds(phase, ph, big, 0, whole, 1) +
                                   rounds(phase, ph, big, whole, ph.tiles, n) + 4 +
                                   JOIN[ph.g[0].words - 1] * n * rest * side * side;
          if (us < least) {
            least = us;
            best.big = big;
            best.ph = ph;
            best.ph.splits = n;
            best.ph.whole = n == 1 ? ph.tiles : whole;
            best.us = us;
          }
        }
    }
    const int64_t rest = best.ph.tiles - best.ph.whole;
    best.ph.base = base;
    if (rest) {   // the parts' room is given back
      const int64_t at = used, side = COSTS[0][best.big].side;
      best.ph.partial = (float*)(base + take(rest * best.ph.splits * side * side * 4));
      used = at;
    }
    return best;
  }

  // The groups' places if a step is shorter by panels than in these launches, or none.
  // (What the plans have taken is taken again: one or the other runs.)
  std::vector<PanelGroup> panels_of(const Plan (&plans)[3]) {
    std::vector<PanelGroup> to;
    double us = 4;
    int blocks = 0;
    used = round_up((int64_t)ORTHO_MATRICES * ORTHO_PARTS * 8, 256);
    for (const OrthoGroup& g : groups) {
      PanelGroup q{};
      q.wide = g.rows <= g.cols;
      q.source_s = std::min(g.rows, g.cols);
      q.source_l = std::max(g.rows, g.cols);
      q.s = (int)round_up(q.source_s, 32);
      q.l = (int)round_up(q.source_l, 32);
      q.first = g.first;
      q.count = g.count;
      q.words = g.words;
      if (q.s > PANEL_SIDE || q.l > PANEL_LENGTH || panel_lds(q) > PANEL_LDS) return {};
      q.per = q.s / PANEL;
      q.block0 = blocks;
      blocks += q.per * q.count;
      to.push_back(q);
    }
    // Rounds of a panel a CU, by the longest of each: 0.8 us a product, and 7.5 a MB of X
    // with a CU alone, 15 where all read (20 with nothing else to wait for).  Fitted to
    // calls of 160 x 160 to 512 x 1024; small launches of tiles take 15% less than their
    // estimate.  Of the 33 steps of profiles/ortho_tiles.csv that either could take, the
    // chosen one is 2.2% behind on the geometric average, 19% at most.
    for (int64_t at = 0; at < blocks; at += 256) {
      double most = 0;
      const double fill = std::min<int64_t>(256, blocks - at) / 256.0;
      for (const PanelGroup& q : to)
        if (q.block0 < at + 256 && q.block0 + (int64_t)q.per * q.count > at) {
          const bool held = panel_held(q);
          const int products = 2 * ((q.s + 255) / 256 + (q.l + 255) / 256);
          most = std::max(most, 0.8 * products + 1e-6 * panel_bytes(q) * (held ? 2 : 4) *
                                                     (7.5 + (held ? 12.5 : 7.5) * fill));
        }
      us += most;
    }
    if (1.15 * us > plans[0].us + plans[1].us + plans[2].us) return {};
    for (PanelGroup& q : to)
      for (int64_t PanelGroup::*at : {&PanelGroup::rows, &PanelGroup::columns,
                                      &PanelGroup::next_rows, &PanelGroup::next_columns})
        q.*at = take((int64_t)q.count * panel_bytes(q));
    return to;
  }
  int run_panels(const char* who, const Scales& sc, int steps, int dest, const OrthoPrep& prep,
                 const std::vector<PanelGroup>& panels, const OrthoOut& out, hipStream_t st) {
    OrthoPanels p{};
    PanelSources first{};
    int blocks = 0, lds = 0;
    bool all = true;
    for (const PanelGroup& q : panels) {
      all = all && panel_held(q);
      p.g[p.groups] = first.g[p.groups] = q;
      first.g[p.groups].parts = prep.g[p.groups].parts;
      ++p.groups;
      blocks += q.per * q.count;
      lds = std::max(lds, panel_lds(q));
    }
    for (int i = 0; i < n; ++i) {
      first.src[i] = prep.src[i];
      first.buf[i] = prep.buf[i];
      first.ld[i] = prep.ld[i];
      first.dt[i] = prep.dt[i];
    }
    first.base = base;
    first.norms = norms;
    first.eps = prep.eps;
    first.scale = prep.scale;
    first.momentum = prep.momentum;
    first.rest = prep.rest;
    first.groups = p.groups;
    first.nesterov = prep.nesterov;
    k_panel_first<<<blocks, PANEL_THREADS, 0, st>>>(first);
    SCAO_LAUNCH_CHECK(who);
    p.base = base;
    for (int k = 0; k < steps; ++k) {
      p.gram = sc.gram[k];
      p.second = sc.second[k];
      p.third = sc.third[k];
      p.a = sc.a[k];
      p.b = sc.b[k];
      p.c = sc.c[k];
      const int to = k + 1 < steps ? ORTHO_NEXT : dest;
      auto* kernel = all ? (to == ORTHO_NEXT     ? k_ortho_panels<true, ORTHO_NEXT>
                            : to == ORTHO_RESULT ? k_ortho_panels<true, ORTHO_RESULT>
                                                 : k_ortho_panels<true, ORTHO_PARAMETER>)
                         : (to == ORTHO_NEXT     ? k_ortho_panels<false, ORTHO_NEXT>
                            : to == ORTHO_RESULT ? k_ortho_panels<false, ORTHO_RESULT>
                                                 : k_ortho_panels<false, ORTHO_PARAMETER>);
      kernel<<<blocks, PANEL_THREADS, lds, st>>>(p, out);
      SCAO_LAUNCH_CHECK(who);
      for (int i = 0; i < p.groups; ++i) {
        std::swap(p.g[i].rows, p.g[i].next_rows);
        std::swap(p.g[i].columns, p.g[i].next_columns);
      }
    }
    return SCAO_OK;
  }

  void prep(OrthoPrep& p, int& blocks) const {
    blocks = 0;
    for (size_t i = 0; i < groups.size(); ++i) {
      const OrthoGroup& g = groups[i];
      OrthoSource& s = p.g[i];
      s.rows = g.rows;
      s.cols = g.cols;
      s.ldx = g.ldx;
      s.first = g.first;
      s.words = g.words;
      s.x = g.x;
      s.x_step = g.x_step;
      s.vecs = 1;
      while (s.vecs < 256 && s.vecs * 8 < g.ldx) s.vecs *= 2;
      s.across = (g.ldx / 8 + s.vecs - 1) / s.vecs;
      const int64_t down = (g.rows + 256 / s.vecs - 1) / (256 / s.vecs), units = down * s.across;
      s.per = (int)std::max<int64_t>(8, (units + ORTHO_PARTS - 1) / ORTHO_PARTS);
      s.parts = (int)((units + s.per - 1) / s.per);
      s.block0 = blocks;
      blocks += s.parts * g.count;
    }
    for (int i = 0; i < n; ++i) {
      const Matrix& e = entry(i);
      p.src[i] = e.src;
      p.buf[i] = e.buf;
      p.ld[i] = (int)e.ld_src;
      p.dt[i] = (uint8_t)e.src_dtype;
    }
    p.groups = (int)groups.size();
    p.base = base;
    p.norms = norms;
  }

  int run(const char* who, const Scales& sc, int steps, double eps, double momentum, bool nesterov,
          int dest, hipStream_t st) {
    Plan plans[3] = {plan(ORTHO_GRAM), plan(ORTHO_SQUARE), plan(ORTHO_UPDATE)};
    const std::vector<PanelGroup> panels = panels_of(plans);
    OrthoPrep p{};
    int blocks;
    prep(p, blocks);
    p.eps = eps;
    p.scale = sc.first;
    p.momentum = (float)momentum;
    p.rest = (float)(1.0 - momentum);
    p.nesterov = nesterov;
    k_ortho_norm<<<blocks, 256, 0, st>>>(p);
    if (panels.empty()) k_ortho_scale<<<blocks, 256, 0, st>>>(p);
    SCAO_LAUNCH_CHECK(who);
    OrthoOut out{};
    for (int i = 0; i < n; ++i) {
      out.p[i] = entry(i).dst;
      out.ld[i] = (int)entry(i).ld_dst;
      out.dt[i] = (uint8_t)entry(i).dst_dtype;
      out.rate[i] = entry(i).rate;
      out.decay[i] = entry(i).decay;
    }
    if (!panels.empty()) return run_panels(who, sc, steps, dest, p, panels, out, st);
    for (int k = 0; k < steps; ++k) {
      plans[ORTHO_GRAM].ph.by = sc.gram[k];
      plans[ORTHO_SQUARE].ph.by = sc.square[k];
      plans[ORTHO_SQUARE].ph.keep = sc.square_keep[k];
      plans[ORTHO_SQUARE].ph.diagonal = sc.diagonal[k];
      plans[ORTHO_UPDATE].ph.by = sc.update[k];
      for (int phase = 0; phase < 3; ++phase) {
        const int to = phase == ORTHO_UPDATE && k + 1 == steps ? dest : ORTHO_NEXT;
        (plans[phase].big ? ortho_tiles256 : ortho_tiles128)(phase, to, plans[phase].ph, out, st);
        SCAO_LAUNCH_CHECK(who);
      }
      for (Plan& q : plans)
        for (int i = 0; i < q.ph.groups; ++i) std::swap(q.ph.g[i].x, q.ph.g[i].y);
    }
    return SCAO_OK;
  }
};

// The matrices in passes, those of one shape together, larger ones first.  A pass
// ends at eight rounds of tiles, so that the workspace does not grow with the model.
constexpr int64_t PASS_TILES = 2048;
template <class F>
int for_passes(const std::vector<Matrix>& m, F&& f) {
  std::vector<int> order;
  for (int i = 0; i < (int)m.size(); ++i)
    if (m[i].rows && m[i].cols) order.push_back(i);
  std::stable_sort(order.begin(), order.end(), [&](int i, int j) {
    const Matrix &a = m[i], &b = m[j];
    if (a.smaller() != b.smaller()) return a.smaller() > b.smaller();
    if (a.rows != b.rows) return a.rows > b.rows;
    return a.cols != b.cols ? a.cols > b.cols : a.words > b.words;
  });
  for (size_t i = 0; i < order.size();) {
    const size_t begin = i;
    int64_t tiles = 0;
    int groups = 0;
    while (i < order.size() && i - begin < ORTHO_MATRICES && tiles < PASS_TILES) {
      const Matrix& e = m[order[i]];
      if ((i == begin || !same_group(e, m[order[i - 1]])) && ++groups > ORTHO_GROUPS) break;
      tiles += e.tiles();
      ++i;
    }
    if (const int rc = f(&order[begin], (int)(i - begin))) return rc;
  }
  return SCAO_OK;
}

bool all_small(const std::vector<Matrix>& m, int steps);
int64_t workspace_of(const std::vector<Matrix>& m, int steps) {
  int64_t most = 0;
  if (all_small(m, steps)) return 0;
  for_passes(m, [&](const int* order, int n) {
    Pass p(m.data(), order, n, nullptr, steps > 1);
    const Plan plans[3] = {p.plan(ORTHO_GRAM), p.plan(ORTHO_SQUARE), p.plan(ORTHO_UPDATE)};
    p.panels_of(plans);
    most = std::max(most, p.peak);
    return SCAO_OK;
  });
  return most;
}

// Whether a workgroup holds every matrix whole: then the call is one launch for up to
// 64 of them.  (Among larger ones small matrices share those's launches.)  A few of
// more than 96 rows are shorter by panels, which share a matrix among workgroups: one of
// 112 x 112 62 us and 48, of 128 x 128 65 and 49, eight 67 and 55, but 32 68 and 75.
bool all_small(const std::vector<Matrix>& m, int steps) {
  if (steps > SMALL_STEPS) return false;
  int n = 0;
  int64_t most = 0;
  for (const Matrix& e : m) {
    if (!e.rows || !e.cols) continue;
    if (e.smaller() > SMALL_SIDE || e.larger() > 4096 ||
        small_lds((int)e.smaller(), (int)e.larger()) > SMALL_LDS)
      return false;
    ++n;
    most = std::max(most, e.smaller());
  }
  return most <= 96 || n > 16;
}
int run_small(const char* who, const std::vector<Matrix>& m, const Scales& sc, int steps, double eps,
              double momentum, bool nesterov, int dest, hipStream_t st) {
  OrthoSmall p{};
  for (int k = 0; k < steps; ++k) {
    p.gram[k] = sc.gram[k];
    p.square[k] = sc.square[k];
    p.keep[k] = sc.square_keep[k];
    p.diagonal[k] = sc.diagonal[k];
    p.update[k] = sc.update[k];
  }
  p.steps = steps;
  p.eps = eps;
  p.scale = sc.first;
  p.momentum = (float)momentum;
  p.rest = (float)(1.0 - momentum);
  p.nesterov = nesterov;
  for (size_t i = 0; i < m.size();) {
    int n = 0, lds = 0;
    for (; i < m.size() && n < ORTHO_MATRICES; ++i) {
      const Matrix& e = m[i];
      if (!e.rows || !e.cols) continue;
      p.src[n] = e.src;
      p.buf[n] = e.buf;
      p.dst[n] = e.dst;
      p.rows[n] = (int)e.rows;
      p.cols[n] = (int)e.cols;
      p.ld_src[n] = (int)e.ld_src;
      p.ld_dst[n] = (int)e.ld_dst;
      p.rate[n] = e.rate;
      p.decay[n] = e.decay;
      p.src_dt[n] = (uint8_t)e.src_dtype;
      p.dst_dt[n] = (uint8_t)e.dst_dtype;
      lds = std::max(lds, small_lds((int)e.smaller(), (int)e.larger()));
      ++n;
    }
    if (!n) break;
    if (dest == ORTHO_RESULT) k_ortho_small<ORTHO_RESULT><<<n, SMALL_THREADS, lds, st>>>(p);
    else k_ortho_small<ORTHO_PARAMETER><<<n, SMALL_THREADS, lds, st>>>(p);
    SCAO_LAUNCH_CHECK(who);
  }
  return SCAO_OK;
}

int run_all(const char* who, const std::vector<Matrix>& m, const double* coefficients, int steps,
            double eps, double momentum, bool nesterov, int dest, void* workspace,
            void* stream) {
  Scales sc;
  SCAO_CHECK_ARG(scales_of(coefficients, steps, sc),
                 "%s: with these coefficients singular values may grow beyond 1024", who);
  if (all_small(m, steps))
    return run_small(who, m, sc, steps, eps, momentum, nesterov, dest, (hipStream_t)stream);
  SCAO_CHECK_ARG((uintptr_t)workspace % 16 == 0, "%s: workspace is not aligned", who);
  return for_passes(m, [&](const int* order, int n) -> int {
    SCAO_CHECK_ARG(workspace, "%s: null workspace", who);
    Pass p(m.data(), order, n, (char*)workspace, steps > 1);
    return p.run(who, sc, steps, eps, momentum, nesterov, dest, (hipStream_t)stream);
  });
}

int check_scheme(const char* who, int n, const void* table, const double* coefficients, int steps,
                 double eps) {
  SCAO_CHECK_ARG(n >= 0 && (n == 0 || table), "%s: null table or negative count", who);
  SCAO_CHECK_ARG(steps >= 1 && steps <= MAX_STEPS, "%s: %d steps (1 to %d)", who, steps, MAX_STEPS);
  SCAO_CHECK_ARG(coefficients, "%s: null coefficients", who);
  for (int i = 0; i < 3 * steps; ++i)
    SCAO_CHECK_ARG(std::isfinite(coefficients[i]), "%s: coefficient %d is no finite number", who, i);
  // (1 / eps has to be a number: a matrix of zeros is one of zeros)
  SCAO_CHECK_ARG(eps >= 1e-300 && std::isfinite(eps), "%s: eps %g (finite, at least 1e-300)", who,
                 eps);
  return SCAO_OK;
}
int check_sizes(const char* who, int i, int64_t rows, int64_t cols, int precision) {
  SCAO_CHECK_ARG(rows >= 0 && cols >= 0 && std::max(rows, cols) < MAX_SIDE &&
                     std::min(rows, cols) <= MAX_SMALLER,
                 "%s: matrix %d is %lld x %lld (sides below 2^20, the smaller one up to 2^15)", who,
                 i, (long long)rows, (long long)cols);
  SCAO_CHECK_ARG(precision == SCAO_ORTHO_FAST || precision == SCAO_ORTHO_FP32,
                 "%s: precision %d of matrix %d", who, precision, i);
  return SCAO_OK;
}
int check_matrix(const char* who, int i, const char* name, const void* p, int64_t rows, int64_t cols,
                 int64_t ld, int dtype) {
  SCAO_CHECK_ARG(dtype >= 0 && dtype <= SCAO_F16, "%s: dtype %d of matrix %d", who, dtype, i);
  SCAO_CHECK_ARG(p && (uintptr_t)p % size_of(dtype) == 0,
                 "%s: %s of matrix %d is null or not aligned to its elements", who, name, i);
  SCAO_CHECK_ARG(rows == 1 || (ld >= cols && ld <= 0x7fffffff),
                 "%s: row stride %lld of %s of matrix %d (%lld columns)", who, (long long)ld, name,
                 i, (long long)cols);
  return SCAO_OK;
}

// Words of an element.  Up to 128 rows or columns two in any case: a tile's beginning
// and end are most of such a product, and one word's roundings spread over the fewer
// singular values (results of 64 x 64 1.5e-3 off, of 1024 x 1024 1.2e-3).
int words_of(int precision, int64_t rows, int64_t cols) {
  return precision == SCAO_ORTHO_FP32 || std::min(rows, cols) <= 128 ? 2 : 1;
}

// what a call writes may not be what it writes or reads elsewhere
struct Range {
  uintptr_t begin, end;
  bool written;
};
int check_apart(const char* who, std::vector<Range>& r) {
  std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
  // the furthest end so far of what is written, and of anything
  uintptr_t wrote = 0, any = 0;
  for (const Range& x : r) {
    SCAO_CHECK_ARG(x.begin >= wrote && (!x.written || x.begin >= any),
                   "%s: two matrices share memory that is written", who);
    any = std::max(any, x.end);
    if (x.written) wrote = std::max(wrote, x.end);
  }
  return SCAO_OK;
}
Range range_of(const void* p, int64_t rows, int64_t cols, int64_t ld, int dtype, bool written) {
  const uintptr_t at = (uintptr_t)p;
  return {at, at + ((rows - 1) * (rows == 1 ? 0 : ld) + cols) * size_of(dtype), written};
}

int collect(const char* who, const scao_ortho_desc* t, int n, bool pointers, std::vector<Matrix>& m) {
  std::vector<Range> r;
  for (int i = 0; i < n; ++i) {
    if (int rc = check_sizes(who, i, t[i].rows, t[i].cols, t[i].precision)) return rc;
    if (pointers && t[i].rows && t[i].cols) {
      if (int rc = check_matrix(who, i, "src", t[i].src, t[i].rows, t[i].cols, t[i].ld_src,
                                t[i].src_dtype))
        return rc;
      if (int rc = check_matrix(who, i, "dst", t[i].dst, t[i].rows, t[i].cols, t[i].ld_dst,
                                t[i].dst_dtype))
        return rc;
      r.push_back(range_of(t[i].src, t[i].rows, t[i].cols, t[i].ld_src, t[i].src_dtype, false));
      r.push_back(range_of(t[i].dst, t[i].rows, t[i].cols, t[i].ld_dst, t[i].dst_dtype, true));
    }
    const int64_t one = t[i].cols;   // a single row's stride is never used
    m.push_back({t[i].src, nullptr, t[i].dst, t[i].rows, t[i].cols,
                 t[i].rows == 1 ? one : t[i].ld_src, t[i].rows == 1 ? one : t[i].ld_dst,
                 t[i].src_dtype, t[i].dst_dtype, 0.f, 0.f,
                 words_of(t[i].precision, t[i].rows, t[i].cols)});
  }
  return check_apart(who, r);
}
int collect(const char* who, const scao_muon_desc* t, int n, bool pointers, std::vector<Matrix>& m) {
  std::vector<Range> r;
  for (int i = 0; i < n; ++i) {
    const auto [rows, cols] = std::pair(t[i].rows, t[i].cols);
    if (int rc = check_sizes(who, i, rows, cols, t[i].precision)) return rc;
    if (pointers && rows && cols) {
      if (int rc = check_matrix(who, i, "p", t[i].p, rows, cols, cols, t[i].dtype)) return rc;
      if (int rc = check_matrix(who, i, "g", t[i].g, rows, cols, cols, t[i].grad_dtype)) return rc;
      if (int rc = check_matrix(who, i, "m", t[i].m, rows, cols, cols, SCAO_F32)) return rc;
      SCAO_CHECK_ARG(std::isfinite(t[i].rate) && std::isfinite(t[i].decay),
                     "%s: rate or decay of matrix %d is no finite number", who, i);
      r.push_back(range_of(t[i].g, rows, cols, cols, t[i].grad_dtype, false));
      r.push_back(range_of(t[i].p, rows, cols, cols, t[i].dtype, true));
      r.push_back(range_of(t[i].m, rows, cols, cols, SCAO_F32, true));
    }
    m.push_back({t[i].g, t[i].m, t[i].p, rows, cols, cols, cols, t[i].grad_dtype, t[i].dtype,
                 t[i].rate, t[i].decay, words_of(t[i].precision, rows, cols)});
  }
  return check_apart(who, r);
}
}  // namespace

namespace {
// no C++ exception leaves a C entry
template <class T, class F>
T guarded(const char* who, int n, T failed, F&& f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    scao_set_error("%s: no host memory for %d matrices", who, n);
    return failed;
  }
}
}  // namespace

extern "C" int64_t scao_orthogonalize_workspace(const scao_ortho_desc* matrices, int n, int steps) {
  const char* who = "scao_orthogonalize_workspace";
  return guarded<int64_t>(who, n, 0, [&]() -> int64_t {
    std::vector<Matrix> m;
    if (n <= 0 || !matrices || collect(who, matrices, n, false, m)) return 0;
    return workspace_of(m, steps);
  });
}

extern "C" int scao_orthogonalize(const scao_ortho_desc* matrices, int n,
                                  const double* coefficients, int steps, double eps,
                                  void* workspace, void* stream) {
  const char* who = "scao_orthogonalize";
  return guarded<int>(who, n, SCAO_ERR_INVALID, [&]() -> int {
    if (int rc = check_scheme(who, n, matrices, coefficients, steps, eps)) return rc;
    std::vector<Matrix> m;
    if (int rc = collect(who, matrices, n, true, m)) return rc;
    return run_all(who, m, coefficients, steps, eps, 0.0, false, ORTHO_RESULT,
                   workspace, stream);
  });
}

extern "C" int64_t scao_muon_workspace(const scao_muon_desc* matrices, int n, int steps) {
  const char* who = "scao_muon_workspace";
  return guarded<int64_t>(who, n, 0, [&]() -> int64_t {
    std::vector<Matrix> m;
    if (n <= 0 || !matrices || collect(who, matrices, n, false, m)) return 0;
    return workspace_of(m, steps);
  });
}

extern "C" int scao_muon_step(const scao_muon_desc* matrices, int n, double momentum, int nesterov,
                              const double* coefficients, int steps, double eps,
                              void* workspace, void* stream) {
  const char* who = "scao_muon_step";
  return guarded<int>(who, n, SCAO_ERR_INVALID, [&]() -> int {
    if (int rc = check_scheme(who, n, matrices, coefficients, steps, eps)) return rc;
    SCAO_CHECK_ARG(momentum >= 0 && momentum < 1, "%s: momentum %g is not in [0, 1)", who, momentum);
    std::vector<Matrix> m;
    if (int rc = collect(who, matrices, n, true, m)) return rc;
    return run_all(who, m, coefficients, steps, eps, momentum, nesterov != 0,
                   ORTHO_PARAMETER, workspace, stream);
  });
}
