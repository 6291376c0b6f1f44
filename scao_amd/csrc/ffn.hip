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
  // The user's matrix itself where it can be, else a packed copy.
  Operand operand(const void* p, int64_t ld, int64_t rows, int64_t cols) {
    if (direct(p, ld, rows, cols)) return Operand{p, rows == 1 ? cols : ld, 0};
    Operand o;
    o.ld = round_up(cols, 8);
    o.plane = rows * o.ld;
    o.p = ws.take(parts * o.plane * 2);
    if (!dry)
      launchers(s.dtype).pack(p, ld, rows, (int)cols, const_cast<void*>(o.p), (int)o.ld, o.plane,
                              st);
    return o;
  }

  // Tile and parts of k for an M x N product of `steps` k steps: the least
  // estimated time.  us of a step with one workgroup a CU and with all a CU
  // holds, and of a tile's beginning and end, fitted to the times of every tile
  // and part count of 225 products (8 to 4096 tokens, 256 x 704 to 4096 x 14336):
  // the choice is 1.7% slower than the best on the geometric average, 17% at
  // most.  For example dx of 24 tokens, 2048 x 8192: 32 x 128 tiles in one part
  // 116 us, in 16 parts 21.8; of 4096 tokens: 256 x 256 in one part 285, in two
  // 183, 128 x 128 in one 251.
  static void choose(int64_t M, int64_t N, int64_t steps, bool gated, bool tokens, int& tile,
                     int& splits) {
    struct Cost {
      int slots;
      double lone, full, ends;
    };
    static const Cost costs[FFN_TILES] = {
        {256, 1.15, 1.50, 4.9}, {512, 0.62, 1.14, 5.2}, {512, 0.56, 0.70, 3.0}, {768, 0.44, 0.96, 1.7}};
    double best = 1e30;
    for (int t = 0; t < (tokens ? FFN_TILES : FFN_64x128); ++t) {
      const Cost& c = costs[t];
      const int64_t cols = gated ? FFN_BN[t] / 2 : FFN_BN[t];
      const int64_t tiles = ((M + FFN_BM[t] - 1) / FFN_BM[t]) * ((N + cols - 1) / cols);
      for (int64_t n : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
        if (n > 1 && (n * 2 > steps || tiles * n > 2048)) break;
        const int64_t per = (steps + n - 1) / n, groups = tiles * n;
        const int64_t rounds = groups / c.slots, rest = groups % c.slots;
        double us = rounds * (per * c.full + c.ends);
        if (rest) {
          const double crowd = c.slots == 256 ? rest / 256.0
                               : rest <= 256  ? 0.0
                                              : (rest - 256.0) / (c.slots - 256.0);
          us += per * (c.lone + (c.full - c.lone) * crowd) + c.ends;
        }
        // the join: a launch, and 8 bytes a part and element
        if (n > 1) us += 2 + 8 / 7.4e6 * n * (double)M * N * (gated ? 2 : 1);
        if (us < best) {
          best = us;
          tile = t;
          splits = (int)n;
        }
      }
    }
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

  int product(int kind, FfnOperands& o, FfnEpilogue& e) {
    const bool gated = kind == FFN_GATE_UP;
    const int64_t steps = (int64_t)o.nseg * ((o.K + FFN_BK - 1) / FFN_BK);
    int tile = 0;
    choose(o.M, o.N, steps, gated, kind != FFN_DW, tile, o.splits);
    const int cols = gated ? FFN_BN[tile] / 2 : FFN_BN[tile];
    o.tiles_m = (o.M + FFN_BM[tile] - 1) / FFN_BM[tile];
    o.tiles_n = (o.N + cols - 1) / cols;
    e.partial = nullptr;
    if (o.splits > 1) {
      const int64_t at = ws.used;   // given back: the next product may write it
      e.partial = (float*)ws.take((int64_t)o.splits * o.tiles_m * o.tiles_n * FFN_BM[tile] *
                                  FFN_BN[tile] * 4);
      peak = std::max(peak, ws.used);
      ws.used = at;
    }
    if (dry) return SCAO_OK;
    launchers(s.dtype).product(kind, tile, o, e, st);
    return SCAO_OK;
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

  // Whether the forward pass alone goes without tiles.  bf16, 2048 x 8192: 8
  // tokens 30 us against 32, 16 tokens 35 against 33; 4096 x 14336: 4 tokens 73
  // against 78, 16 tokens 93 against 79.  The tiles' operands have to be packed
  // in fp32 and where rows begin off 16 bytes, which takes longer than the
  // product: fp32, 4096 x 14336, 64 tokens 394 us against 789.
  bool few() const {
    if (s.tokens <= 8) return true;
    return s.tokens <= FFN_FEW_TOKENS &&
           !(direct(s.w_gate, s.ld_gate, s.f, s.d) && direct(s.w_up, s.ld_up, s.f, s.d) &&
             direct(s.w_down, s.ld_down, s.d, s.f));
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
    Operand g = operand(s.w_gate, s.ld_gate, s.f, s.d), u = operand(s.w_up, s.ld_up, s.f, s.d);
    if (g.ld != u.ld) pair(g, u);
    const Operand down = operand(s.w_down, s.ld_down, s.d, s.f);
    Operand h;
    h.ld = fp;
    h.plane = s.tokens * fp;
    h.p = save ? saved : ws.take(h_bytes());
    FfnOperands o{};
    o.M = (int)s.tokens;
    o.N = (int)s.f;
    o.K = (int)s.d;
    o.lda = x.ld;
    o.ldb = g.ld;
    const void* pu[FFN_MAX_SEG];
    o.nseg = segments(parts, x, 0, g, o.a, o.b);
    segments(parts, x, 0, u, pu, o.b + FFN_MAX_SEG / 2);
    FfnEpilogue e = kept(const_cast<void*>(h.p), save && saved ? (char*)saved + h_bytes() : nullptr,
                         fp);
    if (int rc = product(FFN_GATE_UP, o, e)) return rc;
    o = FfnOperands{};
    o.M = (int)s.tokens;
    o.N = (int)s.d;
    o.K = (int)s.f;
    o.lda = h.ld;
    o.ldb = down.ld;
    o.nseg = segments(parts, h, 0, down, o.a, o.b);
    e = store(y, s.tokens, s.d);
    return product(FFN_DOWN, o, e);
  }

  // gate and up weights with one row stride
  void pair(Operand& g, Operand& u) {
    const int64_t ld = round_up(s.d, 8);
    auto packed = [&](const void* p, int64_t from, Operand& o) {
      if (o.ld == ld && o.p != p) return;
      o.ld = ld;
      o.plane = s.f * ld;
      o.p = ws.take(parts * o.plane * 2);
      if (!dry) launchers(s.dtype).pack(p, from, s.f, (int)s.d, const_cast<void*>(o.p), (int)ld,
                                        o.plane, st);
    };
    packed(s.w_gate, s.ld_gate, g);
    packed(s.w_up, s.ld_up, u);
  }

  int backward(const void* dy_, int64_t ld_dy, const void* saved, void* dx, void* dgate, void* dup,
               void* ddown, bool all) {
    const bool need_w = all || dgate || dup, need_x = all || dx;
    const Operand dy = operand(dy_, ld_dy, s.tokens, s.d);
    Operand h;
    h.p = saved;
    h.ld = fp;
    h.plane = s.tokens * fp;
    if (all || ddown) {
      FfnOperands o{};
      o.M = (int)s.d;
      o.N = (int)s.f;
      o.K = (int)s.tokens;
      o.lda = dy.ld;
      o.ldb = h.ld;
      o.nseg = segments(parts, dy, 0, h, o.a, o.b);
      FfnEpilogue e = store(ddown, s.d, s.f);
      if (int rc = product(FFN_DW, o, e)) return rc;
    }
    if (!need_w && !need_x) return SCAO_OK;
    const Operand down = operand(s.w_down, s.ld_down, s.d, s.f);
    Operand dab;   // da in the first fp columns, db in the others
    dab.ld = 2 * fp;
    dab.plane = s.tokens * dab.ld;
    dab.p = ws.take(parts * dab.plane * 2);
    {
      FfnOperands o{};
      o.M = (int)s.tokens;
      o.N = (int)s.f;
      o.K = (int)s.d;
      o.lda = dy.ld;
      o.ldb = down.ld;
      o.nseg = segments(parts, dy, 0, down, o.a, o.b);
      FfnEpilogue e = kept(const_cast<void*>(dab.p),
                           saved ? (char*)const_cast<void*>(saved) + h_bytes() : nullptr, 2 * fp);
      if (int rc = product(FFN_DH, o, e)) return rc;
    }
    if (need_w) {
      const Operand x = operand(s.x, s.ldx, s.tokens, s.d);
      FfnOperands o{};
      const bool gate = all || dgate, up = all || dup;
      const int64_t from = gate ? 0 : fp;
      o.M = (int)((gate && up ? fp : 0) + s.f);
      o.N = (int)s.d;
      o.K = (int)s.tokens;
      o.lda = dab.ld;
      o.ldb = x.ld;
      o.nseg = segments(parts, dab, from, x, o.a, o.b);
      FfnEpilogue e = store(gate ? dgate : dup, s.f, s.d);
      e.out2 = dup;
      e.second = gate && up ? (int)fp : 0x7fffffff;
      if (int rc = product(FFN_DW, o, e)) return rc;
    }
    if (need_x) {
      Operand g = operand(s.w_gate, s.ld_gate, s.f, s.d), u = operand(s.w_up, s.ld_up, s.f, s.d);
      if (g.ld != u.ld) pair(g, u);
      FfnOperands o{};
      o.M = (int)s.tokens;
      o.N = (int)s.d;
      o.K = (int)s.f;
      o.lda = dab.ld;
      o.ldb = g.ld;
      o.nseg = segments(parts, dab, 0, g, o.a, o.b);
      o.nseg += segments(parts, dab, fp, u, o.a + o.nseg, o.b + o.nseg);
      FfnEpilogue e = store(dx, s.tokens, s.d);
      if (int rc = product(FFN_DX, o, e)) return rc;
    }
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
  SCAO_CHECK_ARG((rows == 1 || ld >= cols) && ld < ((int64_t)1 << 21),
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
                                               int64_t ld_dy) {
  if (check_inputs("scao_ffn_backward_workspace", d)) return 0;
  Block b(*d, nullptr, nullptr, true);
  b.backward(dy, ld_dy, nullptr, nullptr, nullptr, nullptr, nullptr, true);
  return b.need();
}

extern "C" int scao_ffn_backward(const scao_ffn_desc* d, const void* dy, int64_t ld_dy,
                                 const void* saved, void* dx, void* dw_gate, void* dw_up,
                                 void* dw_down, void* workspace, void* stream) {
  const char* who = "scao_ffn_backward";
  if (int rc = check_inputs(who, d)) return rc;
  if (int rc = check_matrix(who, "dy", dy, ld_dy, d->tokens, d->d, d->dtype)) return rc;
  SCAO_CHECK_ARG(saved && workspace && (uintptr_t)saved % 16 == 0 && (uintptr_t)workspace % 16 == 0,
                 "%s: saved or workspace is null or not aligned", who);
  for (void* p : {dx, dw_gate, dw_up, dw_down})
    SCAO_CHECK_ARG((uintptr_t)p % size_of(d->dtype) == 0, "%s: a gradient is not aligned", who);
  Block b(*d, workspace, stream, false);
  if (int rc = b.backward(dy, ld_dy, saved, dx, dw_gate, dw_up, dw_down, false)) return rc;
  SCAO_LAUNCH_CHECK(who);
  return SCAO_OK;
}
