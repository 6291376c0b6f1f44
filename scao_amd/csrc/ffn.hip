// The gated feed-forward block: argument checks, memory plans and the order of
// the launches.  The kernels are in ffn_kernels.hpp and ffn_gemm.hpp.
#include <algorithm>

#include "ffn_few.hpp"

using namespace scao;

namespace {

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
int size_of(int dt) { return dt == SCAO_F32 ? 4 : 2; }

// Pieces of one buffer, 256-byte aligned.  With a null base it only counts.
struct Arena {
  char* base;
  int64_t used = 0;
  explicit Arena(void* b) : base((char*)b) {}
  void* take(int64_t bytes) {
    char* p = base ? base + used : nullptr;
    used += round_up(bytes, 256);
    return p;
  }
};

// A matrix as the products take it: 16-bit elements, one plane or (fp32) the
// three parts, rows of ld elements (a multiple of 8), 16-byte aligned.
struct Operand {
  const void* p = nullptr;
  int64_t ld = 0, plane = 0;
  const void* part(int i, int64_t at = 0) const { return (const uint16_t*)p + i * plane + at; }
};

FfnLaunchers launchers(int dtype) {
  return dtype == SCAO_F32 ? ffn_f32() : dtype == SCAO_BF16 ? ffn_bf16() : ffn_f16();
}

struct Block {
  const scao_ffn_desc& s;
  hipStream_t st;
  Arena ws;
  bool dry;                 // counting only: nothing is launched
  int parts;                // planes of an operand
  int64_t fp;               // columns of h, da and db, with their padding

  Block(const scao_ffn_desc& d, void* workspace, void* stream, bool count)
      : s(d), st((hipStream_t)stream), ws(workspace), dry(count),
        parts(d.dtype == SCAO_F32 ? 3 : 1), fp(round_up(d.f, 8)) {}

  // whether a matrix's rows can be loaded 16 bytes at a time
  bool direct(const void* p, int64_t ld, int64_t rows, int64_t cols) const {
    return s.dtype != SCAO_F32 && (uintptr_t)p % 16 == 0 && (ld % 8 == 0 || rows == 1) &&
           cols % 8 == 0;
  }
  // The user's matrix itself where it can be, else a copy that pack() makes.
  FfnPack packs{};
  Operand operand(const void* p, int64_t ld, int64_t rows, int64_t cols, bool as_is = true) {
    if (as_is && direct(p, ld, rows, cols)) return Operand{p, rows == 1 ? cols : ld, 0};
    Operand o;
    o.ld = round_up(cols, 8);
    o.plane = rows * o.ld;
    o.p = ws.take(parts * o.plane * 2);
    packs.m[packs.n++] = {p, const_cast<void*>(o.p), ld, o.plane, rows, (int)cols, (int)o.ld,
                          packs.groups};
    packs.groups += (rows * (o.ld / 8) + 255) / 256;
    return o;
  }
  // gate and up weights, with one row stride
  void gate_up(Operand& g, Operand& u) {
    const bool same = s.ld_gate == s.ld_up;
    g = operand(s.w_gate, s.ld_gate, s.f, s.d, same);
    // (either alone may start off 16 bytes: then their strides agree only packed)
    u = operand(s.w_up, s.ld_up, s.f, s.d, same && g.p == s.w_gate);
    if (g.ld != u.ld) g = operand(s.w_gate, s.ld_gate, s.f, s.d, false);
  }
  void pack() {
    if (packs.n && !dry) launchers(s.dtype).pack(packs, st);
  }

  // Estimated us of products on tiles: us of a k step with one workgroup a CU
  // and with all a CU holds, and of a tile's beginning and end, fitted to the
  // times of every tile and part count of 225 products (8 to 4096 tokens, 256 x
  // 704 to 4096 x 14336; 256 x 128 tiles: to 66 forward passes).  On the present
  // kernels the choice is 3.2% slower than the best on the geometric average, 44%
  // (9.2 us for 6.4) at most.  For example dx of 24 tokens, 2048 x 8192: 32 x 128
  // tiles in one part 120 us, in 16 parts 20.0; of 4096 tokens: 256 x 256 in one
  // part 286, in two 185, 128 x 128 in one 248.
  struct Cost {
    int slots;
    double lone, full, ends;
    double step(int64_t groups) const {
      const double crowd = groups >= slots  ? 1.0
                           : slots == 256   ? groups / 256.0
                           : groups <= 256  ? 0.0
                                            : (groups - 256.0) / (slots - 256.0);
      return lone + (full - lone) * crowd;
    }
  };
  struct Shape {
    int kind;
    int64_t M, N, steps;
    bool gated;
    int64_t tiles(int t) const {
      const int64_t cols = gated ? FFN_BN[t] / 2 : FFN_BN[t];
      return ((M + FFN_BM[t] - 1) / FFN_BM[t]) * ((N + cols - 1) / cols);
    }
    // the join: a launch, 8 bytes a part and element, and the epilogue's own
    // `moved`, which a tile's end would overlap better
    double moved;
    double join(int64_t n, double share = 1.0) const {
      return n == 1 ? 0.0 : 2 + (8 / 7.4e6 * n * (gated ? 2 : 1) + moved / 5e6) * M * N * share;
    }
    bool may_split(int t, int64_t n) const {
      return n == 1 || (n * 2 <= steps && tiles(t) * n <= 2048);
    }
  };
  static const Cost& cost(int tile) {
    static const Cost costs[FFN_TILES] = {
        {256, 1.15, 1.50, 4.9}, {256, 0.76, 0.93, 4.5}, {512, 0.62, 1.14, 5.2},
        {512, 0.56, 0.70, 3.0}, {768, 0.44, 0.96, 1.7}};
    return costs[tile];
  }
  // How a product is cut: its tile, how many tiles run in one piece and in how
  // many parts the others.  Either all of them are split, or those that do not
  // fill a last round: 777 tokens, 2048 x 11008, gate and up: 344 tiles on 256
  // CUs, the 88 of the second round in two parts.
  struct Cut {
    int tile = 0, whole = 0, splits = 1;
  };
  static double choose(const Shape& s, Cut& cut) {
    double best = 1e30;
    for (int t = 0; t < (s.kind == FFN_DW ? FFN_64x128 : FFN_TILES); ++t) {
      // 256 x 128 tiles for DOWN: 1024 tokens, 2048 x 8192 bf16, 64 of them in four
      // parts, the forward pass 106 us, with 128 x 128 tiles 112.  In the backward
      // pass they change nothing on average (0.1%), and an epilogue that moves bytes
      // gains from the other 128 x 128 tile on its CU.
      if (t == FFN_256x128 && s.kind != FFN_DOWN) continue;
      const Cost& c = cost(t);
      const int64_t tiles = s.tiles(t);
      for (int64_t n : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
        if (!s.may_split(t, n)) break;
        const int64_t per = (s.steps + n - 1) / n;
        for (int64_t whole : {(int64_t)0, tiles / c.slots * c.slots}) {
          if (whole && (n == 1 || whole == tiles)) continue;
          const int64_t groups = (tiles - whole) * n, last = groups % c.slots;
          // a narrow gated tile's epilogue stores single fragments: 300 tokens,
          // 4096 x 11008 bf16, 120 us on 64 x 128 tiles, 90 without this term and
          // 95 on 256 x 256 tiles
          const double end = c.ends + (s.gated && t >= FFN_64x128 ? 2.5 : 0);
          const double part_end = n == 1 ? end : c.ends;
          double us = whole / c.slots * (s.steps * c.full + end) +
                      groups / c.slots * (per * c.full + part_end) +
                      s.join(n, (double)(tiles - whole) / tiles);
          if (last) us += per * c.step(last) + part_end;
          if (us < best) {
            best = us;
            cut = {t, n == 1 ? (int)tiles : (int)whole, (int)n};
          }
        }
      }
    }
    return best;
  }
  // two products in one launch: `a` workgroups of one length, then as many of
  // the other's as fit where these leave room
  static double choose_pair(const Shape& x, const Shape& y, Cut& cx, Cut& cy) {
    double best = 1e30;
    for (int t : {FFN_256x256, FFN_128x128}) {
      const Cost& c = cost(t);
      for (int64_t n : {1, 2, 4, 8, 16}) {
        if (!x.may_split(t, n)) break;
        for (int64_t m : {1, 2, 4, 8, 16}) {
          if (!y.may_split(t, m)) break;
          int64_t ga = x.tiles(t) * n, gb = y.tiles(t) * m;
          const double step = c.step(ga + gb);
          double a = ((x.steps + n - 1) / n) * step + c.ends, b = ((y.steps + m - 1) / m) * step + c.ends;
          if (a < b) {
            std::swap(a, b);
            std::swap(ga, gb);
          }
          // the first's rounds, its last one on `rest` workgroups' places
          const int64_t rounds = ga / c.slots, rest = ga % c.slots;
          const double lo = rounds * a, hi = rest ? lo + a : lo;
          double us = std::max(hi, (ga * a + gb * b) / c.slots);
          // places for the second's beside and behind them
          while ((int64_t)((us - lo) / b + 1e-9) * (c.slots - rest) +
                     (int64_t)((us - hi) / b + 1e-9) * rest < gb)
            us += 0.25 * b;
          us += x.join(n) + y.join(m);
          if (x.moved && t == FFN_256x256) us *= 1.2;   // see run()
          if (us < best) {
            best = us;
            cx = {t, 0, (int)n};
            cy = {t, 0, (int)m};
          }
        }
      }
    }
    return best;
  }

  // a segment for every product of parts that counts: the small ones first
  static int segments(int parts, const Operand& a, int64_t at_a, const Operand& b,
                      const void** pa, const void** pb) {
    static const int small_first[6][2] = {{1, 1}, {0, 2}, {2, 0}, {0, 1}, {1, 0}, {0, 0}};
    const int n = parts == 3 ? 6 : 1;
    for (int i = 0; i < n; ++i) {
      const int* q = small_first[n == 6 ? i : 5];
      pa[i] = a.part(q[0], at_a);
      pb[i] = b.part(q[1]);
    }
    return n;
  }

  Shape shape(int kind, const FfnOperands& o) const {
    const double bytes = kind == FFN_GATE_UP ? 8 : kind == FFN_DH ? 10 : 0;
    return Shape{kind, o.M, o.N, (int64_t)o.nseg * ((o.K + FFN_BK - 1) / FFN_BK), kind == FFN_GATE_UP,
                 s.dtype == SCAO_F32 ? 2 * bytes : bytes};
  }
  struct Product {
    int kind;
    FfnOperands o;
    FfnEpilogue e;
  };
  // the counts of the tiles of C's rows row0 .. to-1, and room for the parts of a
  // split product
  void cut(Product& p, const Cut& c, int64_t to) {
    FfnOperands& o = p.o;
    const int cols = p.kind == FFN_GATE_UP ? FFN_BN[c.tile] / 2 : FFN_BN[c.tile];
    o.tiles_m = (int)((to - o.row0 + FFN_BM[c.tile] - 1) / FFN_BM[c.tile]);
    o.tiles_n = (o.N + cols - 1) / cols;
    o.splits = c.splits;
    o.whole = c.splits == 1 ? o.tiles() : c.whole;
    p.e.partial = nullptr;
    if (o.whole < o.tiles())
      p.e.partial = (float*)ws.take((int64_t)o.splits * (o.tiles() - o.whole) * FFN_BM[c.tile] *
                                    FFN_BN[c.tile] * 4);
    peak = std::max(peak, ws.used);
  }
  void run(Product& p, const Cut& c, int64_t from, int64_t to) {
    const int64_t at = ws.used;   // the parts' room is given back
    p.o.row0 = (int)from;
    cut(p, c, to);
    ws.used = at;
    if (!dry) launchers(s.dtype).product(p.kind, c.tile, p.o, p.e, st);
  }
  // With few rows left over behind whole tiles of 256 these may go by themselves,
  // on narrow tiles, at the price of reading the weights again: 1030 tokens of
  // 2048 x 8192 119 us against 129, where 1024 fill one round exactly.  Not
  // behind rows that are split many times themselves: 300 tokens of 4096 x 11008
  // fp32 886 us, 256 of them in 8 and 16 parts and 44 apart 973.  (Over 141
  // forward passes of up to 128 rows left gate + up 0.8% and down 0.4% behind the
  // better of both choices.)
  void run(Product& p) {
    const Shape all = shape(p.kind, p.o);
    Cut c, head, tail;
    const double us = choose(all, c);
    const int64_t rows = all.M / 256 * 256, left = all.M - rows;
    if (p.kind != FFN_DW && rows && left && left <= 128) {
      Shape a = all, b = all;
      a.M = rows;
      b.M = left;
      const double again = 2.0 * parts * all.N * p.o.K * p.o.nseg / 4.5e6 * (all.gated ? 2 : 1) /
                           (parts == 3 ? 6 : 1);
      const double apart =
          choose(a, head) + 1.15 * std::max(choose(b, tail), again + 3) + 3;
      if (head.splits <= 6 && 1.03 * apart < us) {
        run(p, head, 0, rows);
        run(p, tail, rows, all.M);
        return;
      }
    }
    run(p, c, 0, all.M);
  }
  // dh or dx, and a dW that does not need it
  void run(Product& p, Product& w) {
    const Shape x = shape(p.kind, p.o), y = shape(w.kind, w.o);
    Cut c, cp, cw;
    // dx goes with its dW where the estimates say so by more than a launch's share
    // (8192 tokens, 4096 x 14336 bf16, the whole pass: 6580 us apart, 6760 in
    // pairs).  dh's epilogue moves bytes: two 128 x 128 tiles on a CU hide half of
    // them behind dWd's products, one 256 x 256 tile none, and large tiles lose in
    // an L2 that holds two working sets.  Of the best of apart and both tiles on
    // 89 backward passes (300 to 8192 tokens, 768 x 2048 to 4096 x 11008) dh is
    // 1.3% slower on average, dx 0.8%.  2048 tokens, 768 x 2048 fp32: dh and dWd
    // apart 276 us, on 128 x 128 tiles 260; 8192 tokens, 2048 x 8192 bf16: apart
    // 1378, on 256 x 256 tiles 1439.
    const double apart = choose(x, c) + choose(y, c) + 3;
    if (1.005 * choose_pair(x, y, cp, cw) > apart + 0.5 * x.moved / 5e6 * x.M * x.N) {
      run(p);
      run(w);
      return;
    }
    const int64_t at = ws.used;
    cut(p, cp, x.M);
    cut(w, cw, y.M);
    ws.used = at;
    if (!dry) launchers(s.dtype).pair(p.kind, cp.tile, p.o, p.e, w.o, w.e, st);
  }
  int64_t peak = 0;
  int64_t need() { return std::max(peak, ws.used); }

  FfnEpilogue store(void* out, int64_t rows, int64_t cols) const {
    FfnEpilogue e{};
    e.out = out;
    e.ldo = cols;
    e.rows = (int)rows;
    e.second = 0x7fffffff;
    e.cols = (int)cols;
    return e;
  }
  // h and the kept a and b
  int64_t h_bytes() const { return round_up(parts * s.tokens * fp * 2, 256); }
  int64_t ab_fi() const { return (s.tokens + 15) / 16; }
  int64_t ab_fj() const { return (s.f + 15) / 16; }
  int64_t saved_bytes() const {
    return h_bytes() + (s.dtype == SCAO_F32 ? ab_bytes<SCAO_F32>(ab_fi(), ab_fj())
                                            : ab_bytes<SCAO_BF16>(ab_fi(), ab_fj()));
  }
  FfnEpilogue kept(void* out, void* ab, int64_t ld) const {
    FfnEpilogue e{};
    e.out = out;
    e.ldo = ld;
    e.plane = s.tokens * ld;
    e.rows = (int)s.tokens;
    e.cols = (int)fp;
    e.fi = (int)ab_fi();
    e.fj = (int)ab_fj();
    e.ab = ab;
    e.act = s.act;
    return e;
  }

  // Whether the forward pass alone goes without tiles: up to 8 tokens, and up to
  // 64 while the block is small.  us without tiles and with them:
  //   bf16  2048 x 8192: 8 tokens 28 and 40, 16: 36 and 40, 24: 43 and 38;
  //         1024 x 2816, 64 tokens: 24 and 26; 4096 x 14336: 4 tokens 78 and 87,
  //         8: 81 and 82, 12: 88 and 81
  //   rows off 16 bytes, which tiles have to pack: 1001 x 2049, 32 tokens 32 and
  //         32; 2049 x 8191: 8 tokens 77 and 85, 12: 86 and 82
  //   fp32, which tiles have to split: 2048 x 8192, 64 tokens 167 and 224
  bool few() const {
    if (s.tokens > FFN_FEW_TOKENS) return false;
    if (s.tokens <= 8 || s.dtype == SCAO_F32) return true;
    const bool as_is = direct(s.w_gate, s.ld_gate, s.f, s.d) &&
                       direct(s.w_up, s.ld_up, s.f, s.d) && direct(s.w_down, s.ld_down, s.d, s.f);
    return s.tokens * s.d * s.f <= (int64_t)1 << (as_is ? 28 : 26);
  }
  // h in the block's type, nothing packed
  int forward_few(void* y) {
    void* h = ws.take(s.tokens * s.f * size_of(s.dtype));
    if (dry) return SCAO_OK;
    FfnFew o{s.x, s.w_gate, s.w_up, s.ldx, s.ld_gate, s.ld_up, (int)s.tokens, (int)s.f, (int)s.d};
    FfnEpilogue e = store(h, s.tokens, s.f);
    e.act = s.act;
    launchers(s.dtype).few(o, e, true, st);
    o = FfnFew{h, s.w_down, nullptr, s.f, s.ld_down, 0, (int)s.tokens, (int)s.d, (int)s.f};
    launchers(s.dtype).few(o, store(y, s.tokens, s.d), false, st);
    return SCAO_OK;
  }

  int forward(void* y, void* saved, bool save) {
    if (!save && few()) return forward_few(y);
    const Operand x = operand(s.x, s.ldx, s.tokens, s.d);
    Operand g, u;
    gate_up(g, u);
    const Operand down = operand(s.w_down, s.ld_down, s.d, s.f);
    Operand h;
    h.ld = fp;
    h.plane = s.tokens * fp;
    h.p = save ? saved : ws.take(h_bytes());
    pack();
    Product p{FFN_GATE_UP};
    p.o.M = (int)s.tokens;
    p.o.N = (int)s.f;
    p.o.K = (int)s.d;
    p.o.lda = x.ld;
    p.o.ldb = g.ld;
    const void* pu[FFN_MAX_SEG];
    p.o.nseg = segments(parts, x, 0, g, p.o.a, p.o.b);
    segments(parts, x, 0, u, pu, p.o.b + FFN_MAX_SEG / 2);
    p.e = kept(const_cast<void*>(h.p), save && saved ? (char*)saved + h_bytes() : nullptr, fp);
    run(p);
    Product q{FFN_DOWN};
    q.o.M = (int)s.tokens;
    q.o.N = (int)s.d;
    q.o.K = (int)s.f;
    q.o.lda = h.ld;
    q.o.ldb = down.ld;
    q.o.nseg = segments(parts, h, 0, down, q.o.a, q.o.b);
    q.e = store(y, s.tokens, s.d);
    run(q);
    return SCAO_OK;
  }

  // grads: SCAO_FFN_DX | ... wanted
  int backward(const void* dy_, int64_t ld_dy, const void* saved, void* dx, void* dgate, void* dup,
               void* ddown, int grads) {
    const bool gate = grads & SCAO_FFN_DGATE, up = grads & SCAO_FFN_DUP;
    const bool want_down = grads & SCAO_FFN_DDOWN, want_x = grads & SCAO_FFN_DX;
    const bool want_dh = gate || up || want_x;
    const Operand dy = operand(dy_, ld_dy, s.tokens, s.d);
    Operand h, down, x, g, u, dab;
    h.p = saved;
    h.ld = fp;
    h.plane = s.tokens * fp;
    if (want_dh) down = operand(s.w_down, s.ld_down, s.d, s.f);
    if (gate || up) x = operand(s.x, s.ldx, s.tokens, s.d);
    if (want_x) gate_up(g, u);
    if (want_dh) {   // da in the first fp columns, db in the others
      dab.ld = 2 * fp;
      dab.plane = s.tokens * dab.ld;
      dab.p = ws.take(parts * dab.plane * 2);
    }
    pack();

    Product wd{FFN_DW}, dh{FFN_DH}, wgu{FFN_DW}, px{FFN_DX};
    wd.o.M = (int)s.d;
    wd.o.N = (int)s.f;
    wd.o.K = (int)s.tokens;
    wd.o.lda = dy.ld;
    wd.o.ldb = h.ld;
    wd.o.nseg = segments(parts, dy, 0, h, wd.o.a, wd.o.b);
    wd.e = store(ddown, s.d, s.f);

    dh.o.M = (int)s.tokens;
    dh.o.N = (int)s.f;
    dh.o.K = (int)s.d;
    dh.o.lda = dy.ld;
    dh.o.ldb = down.ld;
    dh.o.nseg = segments(parts, dy, 0, down, dh.o.a, dh.o.b);
    dh.e = kept(const_cast<void*>(dab.p),
                saved ? (char*)const_cast<void*>(saved) + h_bytes() : nullptr, 2 * fp);

    wgu.o.M = (int)((gate && up ? fp : 0) + s.f);
    wgu.o.N = (int)s.d;
    wgu.o.K = (int)s.tokens;
    wgu.o.lda = dab.ld;
    wgu.o.ldb = x.ld;
    wgu.o.nseg = segments(parts, dab, gate ? 0 : fp, x, wgu.o.a, wgu.o.b);
    wgu.e = store(gate ? dgate : dup, s.f, s.d);
    wgu.e.out2 = dup;
    wgu.e.second = gate && up ? (int)fp : 0x7fffffff;

    px.o.M = (int)s.tokens;
    px.o.N = (int)s.d;
    px.o.K = (int)s.f;
    px.o.lda = dab.ld;
    px.o.ldb = g.ld;
    px.o.nseg = segments(parts, dab, 0, g, px.o.a, px.o.b);
    px.o.nseg += segments(parts, dab, fp, u, px.o.a + px.o.nseg, px.o.b + px.o.nseg);
    px.e = store(dx, s.tokens, s.d);

    if (want_down && want_dh) run(dh, wd);
    else if (want_dh) run(dh);
    else if (want_down) run(wd);
    if ((gate || up) && want_x) run(px, wgu);
    else if (want_x) run(px);
    else if (gate || up) run(wgu);
    return SCAO_OK;
  }
};

// descriptor checks; `who` begins the message
int check(const char* who, const scao_ffn_desc* d) {
  SCAO_CHECK_ARG(d, "%s: null descriptor", who);
  SCAO_CHECK_ARG(d->dtype >= 0 && d->dtype <= SCAO_F16, "%s: dtype %d", who, d->dtype);
  SCAO_CHECK_ARG(d->act >= 0 && d->act <= SCAO_ACT_SIGMOID, "%s: activation %d", who, d->act);
  // tile offsets inside an operand and counts of rows and columns are 32 bits
  const int64_t most = (int64_t)1 << 30;
  SCAO_CHECK_ARG(d->tokens >= 1 && d->tokens < most && d->d >= 1 && d->d < ((int64_t)1 << 21) &&
                     d->f >= 1 && d->f < ((int64_t)1 << 20) &&
                     d->tokens * std::max(d->d, d->f) < ((int64_t)1 << 42),
                 "%s: sizes tokens %lld, d %lld, f %lld", who, (long long)d->tokens,
                 (long long)d->d, (long long)d->f);
  return SCAO_OK;
}
int check_matrix(const char* who, const char* name, const void* p, int64_t ld, int64_t rows,
                 int64_t cols, int dtype) {
  SCAO_CHECK_ARG(p && (uintptr_t)p % size_of(dtype) == 0,
                 "%s: %s is null or not aligned to its elements", who, name);
  // (a single row's stride is never used)
  SCAO_CHECK_ARG(rows == 1 || (ld >= cols && ld < ((int64_t)1 << 21)),
                 "%s: row stride %lld of %s (%lld columns; at most 2^21 - 1)", who, (long long)ld,
                 name, (long long)cols);
  return SCAO_OK;
}
int check_inputs(const char* who, const scao_ffn_desc* d) {
  if (int rc = check(who, d)) return rc;
  if (int rc = check_matrix(who, "x", d->x, d->ldx, d->tokens, d->d, d->dtype)) return rc;
  if (int rc = check_matrix(who, "w_gate", d->w_gate, d->ld_gate, d->f, d->d, d->dtype)) return rc;
  if (int rc = check_matrix(who, "w_up", d->w_up, d->ld_up, d->f, d->d, d->dtype)) return rc;
  return check_matrix(who, "w_down", d->w_down, d->ld_down, d->d, d->f, d->dtype);
}

}  // namespace

extern "C" int64_t scao_ffn_saved_bytes(const scao_ffn_desc* d) {
  if (check("scao_ffn_saved_bytes", d)) return 0;
  return Block(*d, nullptr, nullptr, true).saved_bytes();
}

extern "C" int64_t scao_ffn_forward_workspace(const scao_ffn_desc* d, int save) {
  if (check_inputs("scao_ffn_forward_workspace", d)) return 0;
  Block b(*d, nullptr, nullptr, true);
  b.forward(nullptr, nullptr, save != 0);
  return b.need();
}

extern "C" int scao_ffn_forward(const scao_ffn_desc* d, void* y, void* saved, void* workspace,
                                void* stream) {
  if (int rc = check_inputs("scao_ffn_forward", d)) return rc;
  SCAO_CHECK_ARG(y && (uintptr_t)y % size_of(d->dtype) == 0 && (uintptr_t)saved % 16 == 0 &&
                     (uintptr_t)workspace % 16 == 0,
                 "scao_ffn_forward: y is null, or a buffer is not aligned");
  SCAO_CHECK_ARG(workspace || scao_ffn_forward_workspace(d, saved != nullptr) == 0,
                 "scao_ffn_forward: null workspace");
  Block b(*d, workspace, stream, false);
  if (int rc = b.forward(y, saved, saved != nullptr)) return rc;
  SCAO_LAUNCH_CHECK("scao_ffn_forward");
  return SCAO_OK;
}

extern "C" int64_t scao_ffn_backward_workspace(const scao_ffn_desc* d, const void* dy,
                                               int64_t ld_dy, int grads) {
  if (check_inputs("scao_ffn_backward_workspace", d)) return 0;
  Block b(*d, nullptr, nullptr, true);
  b.backward(dy, ld_dy, nullptr, nullptr, nullptr, nullptr, nullptr, grads);
  return b.need();
}

extern "C" int scao_ffn_backward(const scao_ffn_desc* d, const void* dy, int64_t ld_dy,
                                 const void* saved, void* dx, void* dw_gate, void* dw_up,
                                 void* dw_down, void* workspace, void* stream) {
  const char* who = "scao_ffn_backward";
  if (int rc = check_inputs(who, d)) return rc;
  if (int rc = check_matrix(who, "dy", dy, ld_dy, d->tokens, d->d, d->dtype)) return rc;
  const int grads = (dx ? SCAO_FFN_DX : 0) | (dw_gate ? SCAO_FFN_DGATE : 0) |
                    (dw_up ? SCAO_FFN_DUP : 0) | (dw_down ? SCAO_FFN_DDOWN : 0);
  SCAO_CHECK_ARG(saved && (uintptr_t)saved % 16 == 0 && (uintptr_t)workspace % 16 == 0,
                 "%s: saved is null, or it or workspace not aligned", who);
  SCAO_CHECK_ARG(workspace || scao_ffn_backward_workspace(d, dy, ld_dy, grads) == 0,
                 "%s: null workspace", who);
  for (void* p : {dx, dw_gate, dw_up, dw_down})
    SCAO_CHECK_ARG((uintptr_t)p % size_of(d->dtype) == 0, "%s: a gradient is not aligned", who);
  Block b(*d, workspace, stream, false);
  if (int rc = b.backward(dy, ld_dy, saved, dx, dw_gate, dw_up, dw_down, grads)) return rc;
  SCAO_LAUNCH_CHECK(who);
  return SCAO_OK;
}
