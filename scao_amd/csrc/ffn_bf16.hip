// The gated feed-forward block's kernels for bf16.
#include "ffn_few.hpp"

namespace scao {
FfnLaunchers ffn_bf16() {
  return {launch_product<SCAO_BF16>, launch_pair<SCAO_BF16>, launch_pack<SCAO_BF16>, launch_few<SCAO_BF16>};
}
}  // namespace scao
