// The orthogonalisation's products on one fp16 word an element.
#include "ortho_kernels.hpp"

namespace scao {
void ortho_product1(int big, int phase, int dest, const OrthoPhase& ph, const OrthoOut& out,
                    hipStream_t st) {
  ortho_product<1>(big, phase, dest, ph, out, st);
}
}  // namespace scao
