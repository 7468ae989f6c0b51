// fused_host.h — argument checks and parameters that the fused attention entry points share.
#pragma once
#include <cmath>
#include <cstring>

#include "../../include/attn_bwd_b200.h"
#include "fused_common.cuh"
#include "host_shared.h"

namespace attn_bwd {
namespace fused {

inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Strides of a TMA operand: positive multiples of 8 elements along every extent above 1,
// below the descriptor's 2^40 bytes.
inline bool tma_strides_ok(const int64_t* st, int bs, int heads, int seq) {
  const int n[3] = {bs, heads, seq};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (st[i] <= 0 || st[i] % 8 || st[i] >= (1ll << 38))) return false;
  return true;
}

// Whether every row of such a tensor starts at a multiple of 32 bytes (16 elements).
inline bool wide_rows(const void* x, const int64_t* st, int bs, int heads, int seq) {
  const int n[3] = {bs, heads, seq};
  bool ok = (reinterpret_cast<uintptr_t>(x) & 31u) == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (n[i] <= 1 || st[i] % 16 == 0);
  return ok;
}

inline int check_args(const attn_bwd_fused_t* a) {
  if (!a || a->bs < 0 || a->seq_q < 0 || a->seq_kv < 0 || a->heads < 1 || a->kv_heads < 1 ||
      a->heads % a->kv_heads || a->bs > 65535 || a->heads > 65535 || a->seq_q >= (1 << 30) || a->seq_kv >= (1 << 30))
    return ATTN_BWD_EINVAL;
  // scale and softcap in log2 units, and their ratio, have to be finite fp32 numbers
  if (!(a->scale > 0.f) || !(a->scale < 1e38f) || !(a->softcap >= 0.f) || !(a->softcap < 1e38f)) return ATTN_BWD_EINVAL;
  if (a->softcap > 0.f && !(a->softcap > 1e-30f && double(a->scale) / a->softcap < 1e30)) return ATTN_BWD_EINVAL;
  if (a->prefix_lens && !a->causal) return ATTN_BWD_EINVAL;
  // both or neither; an array of no elements may be null
  if ((a->q_documents == nullptr) != (a->kv_documents == nullptr) &&
      (a->q_documents ? a->seq_kv : a->seq_q) != 0 && a->bs != 0)
    return ATTN_BWD_EINVAL;
  if (a->head_dim != 64 && a->head_dim != 128) return ATTN_BWD_EUNSUPPORTED;
  if (a->dtype != ATTN_BWD_DT_BF16 && a->dtype != ATTN_BWD_DT_FP16) return ATTN_BWD_EUNSUPPORTED;
  if (!tma_strides_ok(a->q_stride, a->bs, a->heads, a->seq_q) ||
      !tma_strides_ok(a->k_stride, a->bs, a->kv_heads, a->seq_kv) ||
      !tma_strides_ok(a->v_stride, a->bs, a->kv_heads, a->seq_kv))
    return ATTN_BWD_EALIGN;
  return ATTN_BWD_OK;
}

inline Params base_params(const attn_bwd_fused_t* a) {
  Params p;
  std::memset(&p, 0, sizeof(p));
  p.bs = a->bs;
  p.sq = a->seq_q;
  p.skv = a->seq_kv;
  p.H = a->heads;
  p.Hkv = a->kv_heads;
  p.G = a->heads / a->kv_heads;
  p.off = a->seq_kv - a->seq_q;
  p.causal = a->causal ? 1 : 0;
  p.has_docs = a->q_documents ? 1 : 0;
  p.scale = a->scale;
  p.scale_log2 = a->scale * kLog2e;
  p.cap_u = a->softcap > 0.f ? a->scale / a->softcap : 0.f;
  p.cap_in = a->softcap > 0.f ? 2.f * kLog2e * a->scale / a->softcap : 0.f;
  p.cap_out = a->softcap * kLog2e;
  if (a->softcap > 0.f) {
    p.cap_inv = 1.f / p.cap_out;
    // cap_out * tanh(u x) = cap_out (u x) (1 + k0 (u x)^2 + k1 (u x)^4 + ..)
    const double u = double(a->scale) / a->softcap;
    double f = double(a->softcap) * 1.4426950408889634 * u;
    p.cap_poly[0] = float(f);
    for (int i = 0; i < 5; ++i) {
      f *= u * u;
      p.cap_poly[i + 1] = float(kTanhPoly[i] * f);
      if (!(fabs(p.cap_poly[i + 1]) < 3e38f)) p.cap_u = INFINITY;
    }
  }
  p.slopes = a->slopes;
  p.prefix = a->prefix_lens;
  p.qdoc = a->q_documents;
  p.kdoc = a->kv_documents;
  p.divG = fast_div(p.G);
  p.splits = 1;
  return p;
}

// Map of a [bs, heads, seq, d] tensor with given element strides in the dimension order
// (d, position, head, batch); the box is 64 elements of `rows` positions of one head.
// seq_first = false: order (d, head, position, batch), box 64 x box_heads x rows.  store: boxes of
// 32 elements instead, for store_rows.
inline bool map_bhsd(CUtensorMap* m, const void* ptr, const int64_t* st, int bs, int heads, int seq, int d, bool f16,
                     int rows, int box_heads, bool seq_first, bool store = false) {
  // an extent of 1 is never stepped over, but its stride must still be a valid one
  const auto stride = [&](int i, int n) { return (cuuint64_t)(n > 1 ? st[i] * 2 : (int64_t)d * 2); };
  const cuuint64_t sb = stride(0, bs), sh = stride(1, heads), ss = stride(2, seq);
  cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)seq, (cuuint64_t)heads, (cuuint64_t)bs};
  cuuint64_t str[3] = {ss, sh, sb};
  cuuint32_t box[4] = {64, (cuuint32_t)rows, (cuuint32_t)box_heads, 1};
  if (!seq_first) {
    dims[1] = (cuuint64_t)heads;
    dims[2] = (cuuint64_t)seq;
    str[0] = sh;
    str[1] = ss;
    box[1] = (cuuint32_t)box_heads;
    box[2] = (cuuint32_t)rows;
  }
  if (store) box[0] = 32;
  return host_make_map(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, ptr, dims, str,
                       box, store ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
}

// Shared memory opt-in of a kernel, and the check that ptxas gave it the registers its split
// between warpgroups adds up to.
inline int prepare_kernel(const void* kern, int smem) {
  cudaFuncAttributes at;
  if (cudaFuncGetAttributes(&at, kern) != cudaSuccess) return ATTN_BWD_ECUDA;
  if (at.numRegs != kLaunchRegs) return ATTN_BWD_EUNSUPPORTED;
  if (at.maxDynamicSharedSizeBytes < smem &&
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return ATTN_BWD_ECUDA;
  return ATTN_BWD_OK;
}

// A launch; after: behind another kernel of the same call, whose end it may overlap (see
// wait_for_previous).  One token over 8191 keys for each of 4 sequences: 33.6 us,
// 35.1 launched the plain way; the backward of 2 x 64 x 96: 30.7 and 33.9.
template <typename... P, typename... A>
int launch_kernel(void (*kern)(P...), dim3 grid, int threads, int smem, cudaStream_t s, bool after, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = s;
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = after ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? ATTN_BWD_OK : ATTN_BWD_ECUDA;
}

}  // namespace fused
}  // namespace attn_bwd
