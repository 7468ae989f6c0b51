// fused_token.cu — the forward kernels for units whose rows all fit one tile (see fused_fwd.cuh).
#include "fused_fwd.cuh"
#include "fused_host.h"

namespace attn_bwd {
namespace fused {

ATTN_BWD_FWD_LAUNCHER(launch_token, true)

}  // namespace fused
}  // namespace attn_bwd
