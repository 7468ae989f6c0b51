// fused_token.cu — the forward kernels for units whose rows all fit one tile (see fused_fwd.cuh).
#include "fused_fwd.cuh"

namespace attn_bwd {
namespace fused {

int launch_token(const FwdParams& f, const FwdMaps& m, int d, bool f16, bool cap, cudaStream_t s) {
  return launch_any<true>(f, m, d, f16, cap, s);
}

}  // namespace fused
}  // namespace attn_bwd
