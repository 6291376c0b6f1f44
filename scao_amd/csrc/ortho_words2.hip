// The orthogonalisation's products on two fp16 words an element.
#include "ortho_kernels.hpp"

namespace scao {
void ortho_product2(int big, int phase, int dest, const OrthoPhase& ph, const OrthoOut& out,
                    hipStream_t st) {
  ortho_product<2>(big, phase, dest, ph, out, st);
}
}  // namespace scao
