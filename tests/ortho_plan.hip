// How the orthogonalisation of updates cuts its products, without a GPU: the plans of
// csrc/ortho.hip.  Built by tests/test_ortho_plan.py.
#include "../scao_amd/csrc/ortho.hip"

void scao_set_error(const char*, ...) {}
namespace scao {
void ortho_tiles128(int, int, const OrthoPhase&, const OrthoOut&, hipStream_t) {}
void ortho_tiles256(int, int, const OrthoPhase&, const OrthoOut&, hipStream_t) {}
}  // namespace scao

// Of every pass: a row for each phase {pass, phase, tile's side, tiles, whole ones, parts of
// the others, matrices, 1 if the steps go by panels}; the estimate in us beside it.  A call
// of small matrices is no pass.  How many rows there are, the first `cap` of them in out.
extern "C" int ortho_plan(const scao_ortho_desc* t, int n, int steps, int32_t* out, double* us,
                          int cap) {
  std::vector<Matrix> m;
  if (collect("ortho_plan", t, n, false, m)) return -1;
  if (all_small(m, steps)) return 0;
  int rows = 0, pass = 0;
  for_passes(m, [&](const int* order, int count) -> int {
    Pass p(m.data(), order, count, nullptr, steps > 1);
    Plan plans[3] = {p.plan(ORTHO_GRAM), p.plan(ORTHO_SQUARE), p.plan(ORTHO_UPDATE)};
    const bool panels = !p.panels_of(plans).empty();
    for (int phase = 0; phase < 3; ++phase, ++rows) {
      if (rows >= cap) continue;
      const OrthoPhase& ph = plans[phase].ph;
      const int32_t row[8] = {pass, phase, plans[phase].big ? 256 : 128, ph.tiles, ph.whole,
                              ph.splits, count, panels};
      __builtin_memcpy(out + 8 * rows, row, sizeof(row));
      us[rows] = plans[phase].us;
    }
    ++pass;
    return SCAO_OK;
  });
  return rows;
}
