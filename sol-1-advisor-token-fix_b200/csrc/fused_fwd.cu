// fused_fwd.cu — C entry point of the fused attention forward: the plan (which rows share a
// tile, how the keys are split), descriptors and launches.
#include "fused_fwd.cuh"
#include "fused_host.h"

using namespace attn_bwd;
using namespace attn_bwd::fused;

namespace attn_bwd {
namespace fused {

// Rows of a tile, units and key splits for a shape.
static FwdParams plan_fwd(const attn_bwd_fused_t* a, int sm_count) {
  FwdParams f;
  std::memset(&f, 0, sizeof(f));
  f.c = base_params(a);
  Params& p = f.c;
  const long long whole = (long long)p.H * ((p.sq + TILE - 1) / TILE);
  const int ppt = p.G <= TILE ? TILE / p.G : 0;
  const long long packed = ppt ? (long long)p.Hkv * ((p.sq + ppt - 1) / ppt) : whole;
  f.packed = p.G > 1 && packed < whole;
  f.pos_per_tile = f.packed ? ppt : TILE;
  // two heads of a group have the same keys and the same masks, so a pair of them wastes
  // nothing at the diagonal; an odd group takes 256 positions of a head instead
  f.pair_heads = !f.packed && p.G % 2 == 0;
  f.head_slots = f.packed ? p.Hkv : f.pair_heads ? p.H / 2 : p.H;
  f.div_slots = fast_div(f.head_slots);
  const int pos_per_unit = f.packed ? 2 * ppt : f.pair_heads ? TILE : 2 * TILE;
  f.blocks_q = (p.sq + pos_per_unit - 1) / pos_per_unit;
  p.n_tiles = (p.skv + TILE - 1) / TILE;
  // Too few units for the GPU: split the keys, two tiles a split at least (below that the
  // join costs more than it saves), and never more tiles than a unit's list holds.
  const long long units = (long long)f.blocks_q * f.head_slots * p.bs;
  long long splits = units > 0 ? sm_count / units : 1;
  if (splits > p.n_tiles / 2) splits = p.n_tiles / 2;
  const long long least = p.has_docs ? (p.n_tiles + kMaxList - 1) / kMaxList : 1;
  if (splits < least) splits = least;
  if (splits < 1) splits = 1;
  p.tiles_per_split = int((p.n_tiles + splits - 1) / splits);
  if (p.tiles_per_split < 1) p.tiles_per_split = 1;
  p.splits = (p.n_tiles + p.tiles_per_split - 1) / p.tiles_per_split;
  if (p.splits < 1) p.splits = 1;
  return f;
}

// Workspace: document ranges of the key tiles, then the splits' outputs and row statistics.
static int64_t range_bytes(const Params& p) {
  return p.has_docs ? ((int64_t)p.bs * p.n_tiles * int64_t(sizeof(DocRange)) + 255) / 256 * 256 : 0;
}
static int64_t part_rows(const Params& p) { return p.splits > 1 ? (int64_t)p.splits * p.bs * p.H * p.sq : 0; }

int64_t fwd_workspace(const attn_bwd_fused_t* a, int sm_count) {
  const FwdParams f = plan_fwd(a, sm_count);
  return range_bytes(f.c) + part_rows(f.c) * (a->head_dim + 1) * 4;
}

template <int D, bool F16, bool CAP, bool BIAS>
static int launch(const FwdParams& f, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                  cudaStream_t stream) {
  using C = FwdCfg<D>;
  auto kern = fwd_kernel<D, F16, CAP, BIAS>;
  const int rc = prepare_kernel(reinterpret_cast<const void*>(kern), C::SMEM_BYTES);
  if (rc) return rc;
  if (f.c.has_docs && f.c.n_tiles > 0) {
    const long long tiles = (long long)f.c.bs * f.c.n_tiles;
    doc_ranges_kernel<<<unsigned((tiles + 7) / 8), 256, 0, stream>>>(f.c.kdoc, f.c.skv, nullptr, 0, f.c.bs,
                                                                    const_cast<DocRange*>(f.c.krange), nullptr);
    if (cudaPeekAtLastError() != cudaSuccess) return ATTN_BWD_ECUDA;
  }
  kern<<<dim3(unsigned(f.blocks_q) * f.head_slots, f.c.bs, f.c.splits), kThreads, C::SMEM_BYTES, stream>>>(q, k, v, f);
  if (cudaPeekAtLastError() != cudaSuccess) return ATTN_BWD_ECUDA;
  if (f.c.splits > 1) {
    const long long rows = (long long)f.c.bs * f.c.H * f.c.sq;
    fwd_join_kernel<D, F16><<<unsigned((rows + 7) / 8), 256, 0, stream>>>(f);
    if (cudaPeekAtLastError() != cudaSuccess) return ATTN_BWD_ECUDA;
  }
  return ATTN_BWD_OK;
}

}  // namespace fused
}  // namespace attn_bwd

extern "C" int attn_bwd_b200_fused_fwd(const attn_bwd_fused_t* a, const void* q, const void* k, const void* v, void* o,
                                       float* lse, void* workspace, int64_t workspace_bytes,
                                       attn_bwd_stream_t stream_) {
  int rc = check_args(a);
  if (rc) return rc;
  if (a->bs == 0 || a->seq_q == 0) return ATTN_BWD_OK;
  if (!q || !o || !lse || (a->seq_kv && (!k || !v))) return ATTN_BWD_EINVAL;
  if (!al16(q) || !al16(k) || !al16(v) || !al16(o)) return ATTN_BWD_EALIGN;
  HostDevice dev;
  if ((rc = host_device(&dev))) return rc;
  FwdParams f = plan_fwd(a, dev.sm_count);
  Params& p = f.c;
  p.err = dev.err;
  f.o = o;
  f.lse = lse;
  if (f.blocks_q > (1 << 30) / f.head_slots || p.splits > 65535) return ATTN_BWD_EINVAL;
  const int64_t need = range_bytes(p) + part_rows(p) * (a->head_dim + 1) * 4;
  if (need) {
    if (!workspace || workspace_bytes < need) return ATTN_BWD_EINVAL;
    if (reinterpret_cast<uintptr_t>(workspace) & 255u) return ATTN_BWD_EALIGN;
    p.krange = static_cast<const DocRange*>(workspace);
    f.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + range_bytes(p));
    f.part_lse = f.part_o + part_rows(p) * a->head_dim;
  }
  const bool f16 = a->dtype == ATTN_BWD_DT_FP16;
  CUtensorMap mq, mk, mv;
  std::memset(&mk, 0, sizeof(mk));
  std::memset(&mv, 0, sizeof(mv));
  if (!map_bhsd(&mq, q, a->q_stride, p.bs, p.H, p.sq, a->head_dim, f16, f.pos_per_tile, f.packed ? p.G : 1, false))
    return ATTN_BWD_ETMAP;
  if (p.skv > 0 &&
      (!map_bhsd(&mk, k, a->k_stride, p.bs, p.Hkv, p.skv, a->head_dim, f16, TILE, 1, true) ||
       !map_bhsd(&mv, v, a->v_stride, p.bs, p.Hkv, p.skv, a->head_dim, f16, TILE, 1, true)))
    return ATTN_BWD_ETMAP;
  if (p.skv == 0) mk = mv = mq;   // never loaded from, only prefetched
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream_);
  const bool cap = a->softcap > 0.f, bias = a->slopes != nullptr;
#define ATTN_BWD_FWD(DD, FF)                                                                          \
  if (a->head_dim == DD && f16 == FF)                                                                \
    return cap ? (bias ? launch<DD, FF, true, true>(f, mq, mk, mv, s) : launch<DD, FF, true, false>(f, mq, mk, mv, s)) \
               : (bias ? launch<DD, FF, false, true>(f, mq, mk, mv, s) : launch<DD, FF, false, false>(f, mq, mk, mv, s));
  ATTN_BWD_FWD(128, false)
  ATTN_BWD_FWD(128, true)
  ATTN_BWD_FWD(64, false)
  ATTN_BWD_FWD(64, true)
#undef ATTN_BWD_FWD
  return ATTN_BWD_EUNSUPPORTED;
}
