// The gated feed-forward block's kernels for fp16.
#include "ffn_few.hpp"

namespace scao {
FfnLaunchers ffn_f16() {
  return {launch_product<SCAO_F16>, launch_pair<SCAO_F16>, launch_pack<SCAO_F16>, launch_few<SCAO_F16>};
}
}  // namespace scao
