// fused_fwd.cu — C entry point of the fused attention forward: the plan (which rows share a
// tile, how the keys are split), descriptors and launches.
#include "fused_fwd.cuh"

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
  // Rows of a group share a tile where that takes fewer tiles (one token over 40000 keys, 80 + 8
  // heads: 43 us, 196 with a tile a head; 77 tokens over 32013 keys: 140 and 173, capped in fp16 with 40 + 8
  // heads 101 and 135), though the rows of whole tiles are written faster.
  f.packed = p.G > 1 && packed < whole;
  f.pos_per_tile = f.packed ? ppt : TILE;
  // two heads of a group have the same keys and the same masks, so a pair of them wastes
  // nothing at the diagonal (16 documents of 640, causal, 10 heads a group: 196 us, 252 with 256
  // positions of a head, which is what an odd group takes; a prompt of 4096: 298 and 307)
  f.pair_heads = !f.packed && p.G % 2 == 0;
  f.head_slots = f.packed ? p.Hkv : f.pair_heads ? p.H / 2 : p.H;
  f.div_slots = fast_div(f.head_slots);
  const int pos_per_unit = f.packed ? 2 * ppt : f.pair_heads ? TILE : 2 * TILE;
  f.blocks_q = (p.sq + pos_per_unit - 1) / pos_per_unit;
  p.n_tiles = (p.skv + TILE - 1) / TILE;
  // Two chains in a CTA where a unit's rows fit one tile and there is more than one key tile (4 tokens
  // over 8191 keys: 33.6 us, 38.8 with one chain).
  f.duo = p.n_tiles > 1 && !f.pair_heads && f.blocks_q == 1 && p.sq <= f.pos_per_tile;
  const int parts = f.duo ? 2 : 1;
  // Too few units for the GPU: the keys are split (one token over 40000 keys: 43 us, 287 without; 77
  // tokens over 32013: 140 and 462), two tiles a split at least (one a split is no faster and
  // leaves more to join), and never more tiles than a unit may have.
  const long long units = (long long)f.blocks_q * f.head_slots * p.bs;
  long long splits = units > 0 ? sm_count / units : 1;
  if (splits > p.n_tiles / 2) splits = p.n_tiles / 2;
  const int most = p.has_docs ? kMaxList : kMaxUnit;
  const long long least = (p.n_tiles + most - 1) / most;
  if (splits < least) splits = least;
  if (splits < 1) splits = 1;
  p.tiles_per_split = int((p.n_tiles + splits - 1) / splits);
  if (p.tiles_per_split < 1) p.tiles_per_split = 1;
  f.cta_splits = (p.n_tiles + p.tiles_per_split - 1) / p.tiles_per_split;
  if (f.cta_splits < 1) f.cta_splits = 1;
  p.splits = f.cta_splits * parts;
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

int launch_fwd(const FwdParams& f, const FwdMaps& m, int d, bool f16, bool cap, cudaStream_t s) {
  return launch_any<false>(f, m, d, f16, cap, s);
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
  const int64_t os[3] = {(int64_t)p.sq * p.H * a->head_dim, a->head_dim, (int64_t)p.H * a->head_dim};
  f.wide = wide_rows(o, os, p.bs, p.H, p.sq);
  f.lse = lse;
  if (f.blocks_q > (1 << 30) / f.head_slots || f.cta_splits > 65535) return ATTN_BWD_EINVAL;
  const int64_t need = range_bytes(p) + part_rows(p) * (a->head_dim + 1) * 4;
  if (need) {
    if (!workspace || workspace_bytes < need) return ATTN_BWD_EINVAL;
    if (reinterpret_cast<uintptr_t>(workspace) & 255u) return ATTN_BWD_EALIGN;
    p.krange = static_cast<const DocRange*>(workspace);
    f.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + range_bytes(p));
    f.part_lse = f.part_o + part_rows(p) * a->head_dim;
  }
  const bool f16 = a->dtype == ATTN_BWD_DT_FP16;
  FwdMaps m;
  if (!map_bhsd(&m.q, q, a->q_stride, p.bs, p.H, p.sq, a->head_dim, f16, f.pos_per_tile, f.packed ? p.G : 1, false) ||
      !map_bhsd(&m.o, o, os, p.bs, p.H, p.sq, a->head_dim, f16, 32, 1, false, true))
    return ATTN_BWD_ETMAP;
  m.k = m.v = m.q;   // without keys: never loaded from, only prefetched
  if (p.skv > 0 &&
      (!map_bhsd(&m.k, k, a->k_stride, p.bs, p.Hkv, p.skv, a->head_dim, f16, TILE, 1, true) ||
       !map_bhsd(&m.v, v, a->v_stride, p.bs, p.Hkv, p.skv, a->head_dim, f16, TILE, 1, true)))
    return ATTN_BWD_ETMAP;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream_);
  const bool cap = a->softcap > 0.f;
  if (p.has_docs && p.n_tiles > 0) {
    const long long tiles = (long long)p.bs * p.n_tiles;
    doc_ranges_kernel<<<unsigned((tiles + 7) / 8), 256, 0, s>>>(p.kdoc, p.skv, nullptr, 0, p.bs,
                                                               const_cast<DocRange*>(p.krange), nullptr);
    if (cudaPeekAtLastError() != cudaSuccess) return ATTN_BWD_ECUDA;
  }
  rc = f.duo ? launch_token(f, m, a->head_dim, f16, cap, s) : launch_fwd(f, m, a->head_dim, f16, cap, s);
  if (rc || p.splits == 1) return rc;
  const long long rows = (long long)p.bs * p.H * p.sq;
  const dim3 grid(unsigned((rows + 7) / 8));
  const auto join = a->head_dim == 128 ? (f16 ? fwd_join_kernel<128, true> : fwd_join_kernel<128, false>)
                                       : (f16 ? fwd_join_kernel<64, true> : fwd_join_kernel<64, false>);
  return launch_kernel(join, grid, 256, 0, s, true, f);
}
