// fused_bwd.cu — C entry point of the fused attention backward: plan, descriptors, launches.
#include "fused_bwd.cuh"
#include "fused_host.h"

using namespace attn_bwd;
using namespace attn_bwd::fused;

namespace attn_bwd {
namespace fused {

int64_t fwd_workspace(const attn_bwd_fused_t* a, int sm_count);   // fused_fwd.cu

static int tiles_of(int n) { return (n + TILE - 1) / TILE; }

// Key tiles are the units of dkv.  Too few of them for the GPU: each unit's (head, query tile)
// items are shared among several CTAs, whose fp32 sums are joined in order (512 queries over 4096 keys,
// 16 + 2 heads: the whole backward takes 96 us, 113 without).
static int dkv_splits(const attn_bwd_fused_t* a, int sm_count) {
  const long long units = (long long)tiles_of(a->seq_kv) * a->kv_heads * a->bs;
  const long long items = (long long)(a->heads / a->kv_heads) * tiles_of(a->seq_q);
  if (units == 0) return 1;
  long long s = sm_count / units;
  if (s > items) s = items;
  const long long least = (items + kMaxUnit - 1) / kMaxUnit;
  if (s < least) s = least;
  if (s <= 1) return 1;
  const long long per = (items + s - 1) / s;
  return int((items + per - 1) / per);   // no split without items
}

struct BwdLayout {
  int sq_pad, splits;
  int64_t stat, part, range, total;   // bytes
};
static BwdLayout layout_bwd(const attn_bwd_fused_t* a, int sm_count) {
  BwdLayout l;
  l.sq_pad = tiles_of(a->seq_q) * TILE;
  l.splits = dkv_splits(a, sm_count);
  l.stat = (int64_t)a->bs * a->heads * l.sq_pad * 4;
  l.part = l.splits > 1 ? (int64_t)l.splits * a->bs * a->kv_heads * a->seq_kv * 2 * a->head_dim * 4 : 0;
  // document ranges of the query tiles and of the key tiles
  l.range = a->q_documents ? (int64_t)a->bs * (tiles_of(a->seq_q) + tiles_of(a->seq_kv)) * int64_t(sizeof(DocRange)) : 0;
  l.total = 2 * l.stat + l.part + l.range;
  return l;
}

}  // namespace fused
}  // namespace attn_bwd

extern "C" int64_t attn_bwd_b200_fused_workspace(const attn_bwd_fused_t* a, int backward) {
  int rc = check_args(a);
  if (rc) return -rc;
  HostDevice dev;
  if ((rc = host_device(&dev))) return -rc;
  if (!backward) return fwd_workspace(a, dev.sm_count);
  return layout_bwd(a, dev.sm_count).total;
}

extern "C" int attn_bwd_b200_fused_bwd(const attn_bwd_fused_t* a, const void* go, const void* q, const void* k,
                                       const void* v, const void* o, const float* lse, void* dq, void* dk, void* dv,
                                       void* workspace, int64_t workspace_bytes, attn_bwd_stream_t stream_) {
  int rc = check_args(a);
  if (rc) return rc;
  if (!tma_strides_ok(a->dq_stride, a->bs, a->heads, a->seq_q) ||
      !tma_strides_ok(a->dk_stride, a->bs, a->kv_heads, a->seq_kv) ||
      !tma_strides_ok(a->dv_stride, a->bs, a->kv_heads, a->seq_kv))
    return ATTN_BWD_EALIGN;
  if (a->bs == 0 || (a->seq_q == 0 && a->seq_kv == 0)) return ATTN_BWD_OK;
  if (a->seq_q && (!go || !q || !o || !lse || !dq)) return ATTN_BWD_EINVAL;
  if (a->seq_kv && (!k || !v || !dk || !dv)) return ATTN_BWD_EINVAL;
  if (!al16(go) || !al16(q) || !al16(k) || !al16(v) || !al16(o) || !al16(dq) || !al16(dk) || !al16(dv))
    return ATTN_BWD_EALIGN;
  if (tiles_of(a->seq_q) > (1 << 30) / a->heads || tiles_of(a->seq_kv) > (1 << 30) / a->kv_heads) return ATTN_BWD_EINVAL;
  // with documents a unit lists its tiles
  if (a->q_documents && (tiles_of(a->seq_q) > kMaxList || tiles_of(a->seq_kv) > kMaxList)) return ATTN_BWD_EUNSUPPORTED;
  if (tiles_of(a->seq_kv) > kMaxUnit) return ATTN_BWD_EUNSUPPORTED;   // of one unit of dq
  HostDevice dev;
  if ((rc = host_device(&dev))) return rc;
  const BwdLayout l = layout_bwd(a, dev.sm_count);
  if (l.total && (!workspace || workspace_bytes < l.total)) return ATTN_BWD_EINVAL;
  if (reinterpret_cast<uintptr_t>(workspace) & 255u) return ATTN_BWD_EALIGN;
  BwdParams f;
  std::memset(&f, 0, sizeof(f));
  f.c = base_params(a);
  f.c.err = dev.err;
  f.c.n_tiles = tiles_of(a->seq_q);
  f.c.splits = l.splits;
  f.sq_pad = l.sq_pad;
  float* ws = static_cast<float*>(workspace);
  f.o = static_cast<const uint8_t*>(o);
  f.lse = lse;
  f.nlse = ws;
  f.ndelta = ws + l.stat / 4;
  f.n_kt = tiles_of(a->seq_kv);
  f.divH = fast_div(a->heads);
  f.divHkv = fast_div(a->kv_heads);
  f.part = ws + l.stat / 2;
  f.c.qrange = reinterpret_cast<const DocRange*>(reinterpret_cast<const uint8_t*>(f.part) + l.part);
  f.c.krange = f.c.qrange + (int64_t)a->bs * f.c.n_tiles;
  f.dk = dk;
  f.dv = dv;
  // an extent of 1 has no stride that counts
  const auto set = [&](long long* dst, const int64_t* src, int heads, int seq) {
    dst[0] = a->bs > 1 ? src[0] : 0;
    dst[1] = heads > 1 ? src[1] : 0;
    dst[2] = seq > 1 ? src[2] : 0;
  };
  set(f.dks, a->dk_stride, a->kv_heads, a->seq_kv);
  set(f.dvs, a->dv_stride, a->kv_heads, a->seq_kv);
  f.wide = wide_rows(dk, a->dk_stride, a->bs, a->kv_heads, a->seq_kv) &&
           wide_rows(dv, a->dv_stride, a->bs, a->kv_heads, a->seq_kv);
  const bool f16 = a->dtype == ATTN_BWD_DT_FP16;
  CUtensorMap mq, md, mk, mv;
  std::memset(&mk, 0, sizeof(mk));
  std::memset(&mq, 0, sizeof(mq));
  mv = mk;
  md = mq;
  const int64_t os[3] = {(int64_t)a->seq_q * a->heads * a->head_dim, a->head_dim, (int64_t)a->heads * a->head_dim};
  if (a->seq_q &&
      (!map_bhsd(&mq, q, a->q_stride, a->bs, a->heads, a->seq_q, a->head_dim, f16, TILE, 1, true) ||
       !map_bhsd(&md, go, os, a->bs, a->heads, a->seq_q, a->head_dim, f16, TILE, 1, true)))
    return ATTN_BWD_ETMAP;
  if (a->seq_kv &&
      (!map_bhsd(&mk, k, a->k_stride, a->bs, a->kv_heads, a->seq_kv, a->head_dim, f16, TILE, 1, true) ||
       !map_bhsd(&mv, v, a->v_stride, a->bs, a->kv_heads, a->seq_kv, a->head_dim, f16, TILE, 1, true)))
    return ATTN_BWD_ETMAP;
  CUtensorMap mdq;
  std::memset(&mdq, 0, sizeof(mdq));
  if (a->seq_q && !map_bhsd(&mdq, dq, a->dq_stride, a->bs, a->heads, a->seq_q, a->head_dim, f16, 32, 1, true, true))
    return ATTN_BWD_ETMAP;
  if (!a->seq_q) mq = md = mk;   // never loaded from, only prefetched
  if (!a->seq_kv) mk = mv = mq;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream_);
  const bool cap = a->softcap > 0.f;
  const int d = a->head_dim;
  if (f.c.has_docs) {
    const long long tiles = (long long)a->bs * (f.c.n_tiles + f.n_kt);
    doc_ranges_kernel<<<unsigned((tiles + 7) / 8), 256, 0, s>>>(f.c.kdoc, a->seq_kv, f.c.qdoc, a->seq_q, a->bs,
                                                                const_cast<DocRange*>(f.c.krange),
                                                                const_cast<DocRange*>(f.c.qrange));
    if (cudaPeekAtLastError() != cudaSuccess) return ATTN_BWD_ECUDA;
  }
  if (a->seq_q && (rc = launch_dq(f, mq, md, mk, mv, mdq, d, f16, cap, s))) return rc;
  if (a->seq_kv && (rc = launch_dkv(f, mq, md, mk, mv, d, f16, cap, s))) return rc;
  return ATTN_BWD_OK;
}
