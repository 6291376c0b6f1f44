// The launches that the feed-forward block plans, without a GPU: csrc/ffn.hip with
// launchers that write them down. Built for the host alone by tests/test_ffn_plan.py.
#include "../scao_amd/csrc/ffn.hip"

#include <vector>

namespace {

struct Launch {   // mirrored in tests/test_ffn_plan.py
  int32_t kind, tile, type, whole, tiles, splits, row0, paired;
};
std::vector<Launch> launches;

template <int TYPE>
void put(int kind, int tile, const FfnOperands& o, bool paired) {
  launches.push_back({kind, tile, TYPE, o.whole, o.tiles(), o.splits, o.row0, paired});
}
template <int TYPE>
FfnLaunchers recorders() {
  return {[](int kind, int tile, const FfnOperands& o, const FfnEpilogue&, hipStream_t) {
            put<TYPE>(kind, tile, o, false);
          },
          [](int kind, int tile, const FfnOperands& a, const FfnEpilogue&, const FfnOperands& b,
             const FfnEpilogue&, hipStream_t) {
            put<TYPE>(kind, tile, a, true);
            put<TYPE>(FFN_DW, tile, b, true);
          },
          [](const FfnPack&, hipStream_t) {},
          [](const FfnFew& o, const FfnEpilogue&, bool gated, hipStream_t) {
            launches.push_back({gated ? -1 : -2, 0, TYPE, 0, o.tokens, o.cols, 0, 0});
          }};
}

}  // namespace

namespace scao {
FfnLaunchers ffn_f32() { return recorders<SCAO_F32>(); }
FfnLaunchers ffn_bf16() { return recorders<SCAO_BF16>(); }
FfnLaunchers ffn_f16() { return recorders<SCAO_F16>(); }
}  // namespace scao

void scao_set_error(const char*, ...) {}

// the forward pass (train: with what it saves, and the backward pass of all
// gradients); how many launches there are, the first `cap` of them in out
extern "C" int ffn_plan(const scao_ffn_desc* d, int train, int64_t ld_dy, int32_t* out, int cap) {
  launches.clear();
  alignas(16) static char at[16];
  Block f(*d, at, nullptr, false);
  f.forward(at, train ? at : nullptr, train);
  if (train) {
    Block b(*d, at, nullptr, false);
    b.backward(at, ld_dy, at, at, at, at, at, 15);
  }
  for (int i = 0; i < (int)launches.size() && i < cap; ++i)
    __builtin_memcpy(out + 8 * i, &launches[i], sizeof(Launch));
  return (int)launches.size();
}

// the choice for one product alone: tile, tiles in one piece, parts of the others,
// tiles in all; the estimate in us
extern "C" double ffn_choose(int kind, int64_t tokens, int64_t d, int64_t f, int32_t* out) {
  scao_ffn_desc s{};
  s.dtype = SCAO_BF16;
  const Block b(s, nullptr, nullptr, true);
  FfnOperands o{};
  const bool over_f = kind == FFN_DOWN || kind == FFN_DX;
  o.M = (int)(kind == FFN_DW ? 2 * f : tokens);
  o.N = (int)(kind == FFN_GATE_UP || kind == FFN_DH ? f : d);
  o.K = (int)(kind == FFN_DW ? tokens : over_f ? f : d);
  o.nseg = kind == FFN_DX ? 2 : 1;
  Block::Cut c;
  const Block::Shape shape = b.shape(kind, o);
  const double us = Block::choose(shape, c);
  out[0] = c.tile;
  out[1] = c.whole;
  out[2] = c.splits;
  out[3] = (int32_t)shape.tiles(c.tile);
  return us;
}
