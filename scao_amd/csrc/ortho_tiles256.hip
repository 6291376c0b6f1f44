// The orthogonalisation's products on 256 x 256 tiles.
#include "ortho_kernels.hpp"

namespace scao {
void ortho_tiles256(int phase, int dest, const OrthoPhase& ph, const OrthoOut& out, hipStream_t st) {
  ortho_launch<256>(phase, dest, ph, out, st);
}
}  // namespace scao
