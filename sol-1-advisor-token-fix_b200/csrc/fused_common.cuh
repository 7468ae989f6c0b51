// fused_common.cuh — what the fused attention kernels share: parameters, which keys a query
// sees, the list of key (or query) tiles a CTA visits, and the score transform.
//
// Scores are kept in units of log2: t = s * log2(e), so that p = 2^(t - t_max).
#pragma once
#include <cuda_fp16.h>

#include "sm100.cuh"

namespace attn_bwd {
namespace fused {
using namespace sm100;

constexpr int TILE = 128;        // rows of a query tile, keys of a key tile
constexpr int kMaxList = 2048;   // tiles that one CTA visits at most
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Params {
  int bs, sq, skv, H, Hkv, G;
  int off;                 // position of query row 0: skv - sq
  int causal, has_docs;
  float scale;             // of the scores
  float scale_log2;        // scale * log2(e)
  float cap_in;            // softcap: 2 * log2(e) * scale / softcap
  float cap_out;           // softcap * log2(e)
  const float* slopes;     // [H] or null
  const int* prefix;       // [bs] or null
  const int *qdoc, *kdoc;  // [bs, sq], [bs, skv] or null
  int n_tiles;             // tiles of the axis a CTA loops over
  int splits, tiles_per_split;
  int* err;
};

// Number of keys (from key 0) that query row `r` of batch row b sees when documents are left
// out of account: a prefix, then causal.  Never above skv; 0 or less: none.
__device__ __forceinline__ int row_limit(const Params& p, int r, int pre) {
  if (!p.causal) return p.skv;
  return min(p.skv, max(r + p.off + 1, pre));
}

// Lowest and highest document number (>= 0) of n ids, and whether any id is negative, over
// one warp; every lane returns the same values.  No id >= 0: lo > hi.
struct DocRange {
  int lo, hi;
  bool neg;
};
__device__ __forceinline__ DocRange warp_doc_range(const int* ids, int n, uint32_t lane) {
  int lo = 0x7fffffff, hi = -1;
  bool neg = false;
  for (int i = int(lane); i < n; i += 32) {
    const int d = __ldg(ids + i);
    if (d < 0) neg = true;
    else {
      lo = min(lo, d);
      hi = max(hi, d);
    }
  }
  DocRange r;
  r.lo = __reduce_min_sync(0xffffffffu, lo);
  r.hi = __reduce_max_sync(0xffffffffu, hi);
  r.neg = __any_sync(0xffffffffu, neg);
  return r;
}

// List entry: tile offset from the CTA's first tile, and whether single scores of the tile
// have to be masked, and whether rows of the streamed tile belong to no document and so are
// cleared before a product reads them.
constexpr uint32_t kEntMask = 0x8000u, kEntScrub = 0x4000u, kEntTile = 0x3fffu;
constexpr int kStSkip = 0, kStFull = 1, kStMask = 2, kStScrub = 4;

// State of the pair (query range, key range): rows of the range [r0, r1], keys [j0, j1].
__device__ __forceinline__ int pair_state(const Params& p, int pre, int r0, int r1, int j0, int j1, bool docs,
                                          const DocRange& qd, const DocRange& kd) {
  const int lim0 = row_limit(p, r0, pre), lim1 = row_limit(p, r1, pre);   // limits grow with the row
  if (lim1 <= j0) return kStSkip;
  bool full = lim0 > j1;
  if (docs) {
    if (qd.hi < qd.lo || kd.hi < kd.lo || qd.hi < kd.lo || kd.hi < qd.lo) return kStSkip;
    full = full && !qd.neg && !kd.neg && qd.lo == qd.hi && kd.lo == kd.hi;
  }
  return full ? kStFull : kStMask;
}

// Turns states[0..n) (shared memory) into the list of tiles that are not skipped; one warp.
__device__ __forceinline__ int compact_list(const uint8_t* states, int n, uint16_t* list, uint32_t lane) {
  int cnt = 0;
  for (int t0 = 0; t0 < n; t0 += 32) {
    const int t = t0 + int(lane);
    const int st = t < n ? states[t] : kStSkip;
    const uint32_t vote = __ballot_sync(0xffffffffu, st != kStSkip);
    if (st != kStSkip)
      list[cnt + __popc(vote & ((1u << lane) - 1u))] =
          uint16_t(uint32_t(t) | ((st & kStMask) ? kEntMask : 0u) | ((st & kStScrub) ? kEntScrub : 0u));
    cnt += __popc(vote);
  }
  return cnt;
}

// Register split of the attention kernels: three warpgroups are launched with 168 registers a
// thread (504 in sum); the two that hold score rows grow to 216, the one that issues copies and
// products shrinks to 72: 216 + 216 + 72 = 504.  The host launches only kernels that ptxas
// gave 168.
constexpr int kLaunchRegs = 168, kThreads = 384;
__device__ __forceinline__ void regs_grow() { asm volatile("setmaxnreg.inc.sync.aligned.u32 216;"); }
__device__ __forceinline__ void regs_shrink() { asm volatile("setmaxnreg.dec.sync.aligned.u32 72;"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <bool F16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if (F16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(bf16lo(w), bf16hi(w));
}

// 1 / (1 + e^(2x)) with 2 x log2(e) given: tanh x = 1 - 2r and tanh' x = 4 r (1 - r), both to
// fp32 accuracy (2^z overflows to inf, whose reciprocal is 0: the limit).
__device__ __forceinline__ float cap_r(float z) { return rcp(1.f + ex2(z)); }

// kind::f16 instruction descriptor for fp16 (0) or bf16 (1) operands, f32 accumulator.
__host__ __device__ constexpr uint32_t idesc16(bool f16, int M, int N, bool a_mn, bool b_mn) {
  return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}
// D[tmem] (+)= A[tmem] * B[smem]^T: A holds 16-bit pairs along K, one 32-bit column a pair.
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

// Product of a K-major A tile [128 x D] and a K-major B tile [128 x D]: D[128 x 128].
// Tiles are D / 64 blocks of [128 rows x 128 bytes], 128-byte swizzled.
template <int D>
__device__ __forceinline__ void mma_kk(uint32_t d_tmem, uint32_t a, uint32_t b, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const uint32_t o = (kk >> 2) * (TILE * 128) + (kk & 3) * 32;
    umma_bf16(d_tmem, sdesc_sw128(a + o, 16, 1024), sdesc_sw128(b + o, 16, 1024), idesc, kk > 0 ? 1u : 0u);
  }
}
// Product of A [128 x 128] in TMEM (columns a0.. for the first 64 of K, a1.. for the second) and a
// tile [128 rows x D] whose rows are K: D[128 x D] (+)=.  kk: steps [k0, k1) of 16 rows.
template <int D>
__device__ __forceinline__ void mma_tn(uint32_t d_tmem, uint32_t a0, uint32_t a1, uint32_t b, uint32_t idesc,
                                       bool accumulate, int k0 = 0, int k1 = 8) {
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) {
    if (kk < k0 || kk >= k1) continue;
    const uint32_t at = (kk < 4 ? a0 : a1) + (kk & 3) * 8;
    umma_ts(d_tmem, at, sdesc_sw128(b + kk * 2048, TILE * 128, 1024), idesc, (accumulate || kk > 0) ? 1u : 0u);
  }
}

// Clears the rows of a [128 x D] tile whose document is negative (or that lie behind the
// end): the tensor cores would turn a NaN there times a probability of 0 into NaN.  One warp;
// the caller has waited for the tile and is the only one to read it.
template <int D>
__device__ __forceinline__ void scrub_rows(uint32_t tile, const int* ids, int n, uint32_t lane) {
  for (int r = 0; r < TILE; ++r) {
    if (r < n && __ldg(ids + r) >= 0) continue;
    if (int(lane) < D / 8) sts128(tile + (lane >> 3) * (TILE * 128) + r * 128 + (lane & 7) * 16, make_uint4(0, 0, 0, 0));
  }
  fence_proxy_async_smem();
  __syncwarp();
}

}  // namespace fused
}  // namespace attn_bwd
