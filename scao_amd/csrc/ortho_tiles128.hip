// The orthogonalisation's products on 128 x 128 tiles.
#include "ortho_kernels.hpp"

namespace scao {
void ortho_tiles128(int phase, int dest, const OrthoPhase& ph, const OrthoOut& out, hipStream_t st) {
  ortho_launch<128>(phase, dest, ph, out, st);
}
}  // namespace scao
