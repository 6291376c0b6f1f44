// The gated feed-forward block's kernels for fp32.
#include "ffn_few.hpp"

namespace scao {
FfnLaunchers ffn_f32() {
  return {launch_product<SCAO_F32>, launch_pair<SCAO_F32>, launch_pack<SCAO_F32>, launch_few<SCAO_F32>};
}
}  // namespace scao
