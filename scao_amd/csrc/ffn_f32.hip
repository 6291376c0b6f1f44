// The gated feed-forward block's kernels for fp32.
#include "ffn_kernels.hpp"

namespace scao {
FfnLaunchers ffn_f32() { return {launch_product<SCAO_F32>, launch_pack<SCAO_F32>}; }
}
