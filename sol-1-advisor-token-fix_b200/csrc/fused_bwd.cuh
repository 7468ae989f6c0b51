// fused_bwd.cuh — attention backward without materialised weights.
//
//   p = 2^(t - lse2)   dv = p^T do   dp = do v^T   ds = p (dp - delta) [tanh']   dq = scale ds k   dk = scale ds^T q
//
// Two kernels that each recompute p and dp, so that neither dq nor dk / dv needs atomics and
// equal inputs give equal bits; together 7 products of a tile pair instead of 5.
//   dkv: one key tile a CTA, streams the query tiles of all heads of the group.  It computes the
//        transposed scores (keys are rows), so p^T and ds^T are A operands in TMEM and the sum over
//        the group's heads happens in the accumulators.
//   dq:  one query tile of one head a CTA, streams the key tiles.  It runs first and leaves the
//        rows' statistics to dkv (delta from the resident do and a read of o; from the weights where
//        the rows have one key tile).
// In both, warp 8 is the TMA producer, warp 9 issues tcgen05, warp 10 fetches units (and makes their
// lists of tiles), and warps 0-7 turn scores into weights: TMEM lane quadrant warp % 4, columns
// 64 * (warp / 4).. of each tile.
//
// What bounds them: neither the tensor cores (active 45 % of the time in dq, 54 % in dkv) nor memory (6 %
// of its rate), but the chain of a tile: scores, weights, ds, product, with 256 threads to hide
// its waits.  4096 x 4096, 80 + 8 heads of 128, bf16: 2150 us without a mask (0.80 PFLOP/s by the five
// products, 1.12 by the seven that are computed), 1030 us causal, in bursts (see fused_fwd.cuh).  Accumulating dq by atomics
// would save two products, and the order of its sums would change from run to run.
#pragma once
#include <type_traits>

#include "fused_common.cuh"

namespace attn_bwd {
namespace fused {

struct BwdParams {
  Params c;
  int sq_pad;            // sq rounded up to tiles: row length of nlse and ndelta
  int n_kt;              // key tiles
  FastDiv divH, divHkv;
  const uint8_t* o;      // [bs, sq, H, D]
  const float* lse;      // [bs, H, sq]
  float* nlse;           // [bs * H, sq_pad]: -lse * log2(e); -inf for rows that see nothing
  float* ndelta;         // [bs * H, sq_pad]: -sum(do * o); dq writes both, dkv reads them
  void *dk, *dv;
  long long dks[3], dvs[3];   // element strides: batch, head, position
  int wide;                   // rows of dk and dv start at multiples of 32 bytes
  float* part;           // dkv, splits > 1: [split][bs * Hkv * skv][2][D], dk first
};

template <int D>
struct BwdCfg {
  static constexpr int TILE_BYTES = TILE * D * 2;
  static constexpr int ST = 4;
  static constexpr int OFF_A = 0;                               // two resident tiles
  static constexpr int OFF_RING = 2 * TILE_BYTES;
  // dkv: 2 x (nlse, ndelta) of 128 rows; dq: 2 x (halves of 128 rows' sums of p dp and p, or of delta)
  static constexpr int OFF_STAT = OFF_RING + ST * TILE_BYTES;
  static constexpr int OFF_STAGE = OFF_STAT + 4 * 2 * TILE * 4;   // 2 KB for each warp of rows
  static constexpr int OFF_LIST = OFF_STAGE + 8 * 2048;
  static constexpr int OFF_UNIT = OFF_LIST + 2 * kMaxList * 2;
  static constexpr int OFF_BAR = OFF_UNIT + 3 * 16;
  static constexpr int NBAR = 3 + 2 * ST + 8 + 6 + 4;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int SMEM_BYTES = OFF_MISC + 16 + 1024;
  static_assert(SMEM_BYTES <= 227 * 1024, "backward kernel shared memory");
};

struct BwdShared {
  uint8_t* smem;
  uint64_t *res_full, *res_empty, *all_done, *full, *empty, *s_full, *p_ready, *dp_full, *ds_ready, *done;
  uint64_t* pair;   // dq: [quadrant] the two warps of its rows
  uint32_t* tmem_slot;
  volatile int* abort_flag;
  uint16_t* lists;
  Scheduler sched;
};
template <int D>
__device__ __forceinline__ BwdShared bwd_shared(uint8_t* raw) {
  using C = BwdCfg<D>;
  BwdShared s;
  s.smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint64_t* b = reinterpret_cast<uint64_t*>(s.smem + C::OFF_BAR);
  s.res_full = b;
  s.res_empty = b + 1;
  s.all_done = b + 2;
  s.full = b + 3;
  s.empty = s.full + C::ST;
  s.s_full = s.empty + C::ST;
  s.p_ready = s.s_full + 2;   // dq: one s_full a score tile
  s.dp_full = s.p_ready + 2;  // p_ready, ds_ready: one for each 32 of a thread's 64 columns
  s.ds_ready = s.dp_full + 1;
  s.done = s.ds_ready + 2;
  s.sched.slot = reinterpret_cast<Unit*>(s.smem + C::OFF_UNIT);
  s.sched.handle = smem_u32(s.smem + C::OFF_UNIT + 32);
  s.sched.full = s.done + 1;
  s.sched.empty = s.sched.full + 2;
  s.sched.answer = s.sched.empty + 2;
  s.sched.ask = s.sched.answer + 1;
  s.pair = s.sched.ask + 1;
  s.tmem_slot = reinterpret_cast<uint32_t*>(s.smem + C::OFF_MISC);
  s.abort_flag = reinterpret_cast<volatile int*>(s.smem + C::OFF_MISC + 4);
  s.lists = reinterpret_cast<uint16_t*>(s.smem + C::OFF_LIST);
  return s;
}
// Barriers, descriptors and TMEM; returns the TMEM base.  res_users: arrivals that free the resident
// tiles.
__device__ __forceinline__ uint32_t bwd_begin(const BwdShared& s, int st, int res_users, const CUtensorMap* q, const CUtensorMap* go,
                                              const CUtensorMap* k, const CUtensorMap* v) {
  const uint32_t warp = warp_id(), lane = lane_id();
  if (threadIdx.x == 0) {
    mbar_init(s.res_full, 1);
    mbar_init(s.res_empty, res_users);
    mbar_init(s.all_done, 1);
    for (int i = 0; i < st; ++i) { mbar_init(&s.full[i], 1); mbar_init(&s.empty[i], 1); }
    mbar_init(&s.s_full[0], 1);
    mbar_init(&s.s_full[1], 1);
    for (int i = 0; i < 2; ++i) { mbar_init(&s.p_ready[i], 8); mbar_init(&s.ds_ready[i], 8); }
    mbar_init(s.dp_full, 1);
    mbar_init(s.done, 1);
    for (int i = 0; i < 4; ++i) mbar_init(&s.pair[i], 2);
    scheduler_init(s.sched);
    *s.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 8 && lane == 0) {
    prefetch_tmap(q);
    prefetch_tmap(go);
    prefetch_tmap(k);
    prefetch_tmap(v);
  }
  if (warp == 9) { tmem_alloc(s.tmem_slot, 512); tmem_relinquish(); }
  wait_for_previous();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  return *s.tmem_slot;
}
__device__ __forceinline__ void bwd_end(const BwdShared& s, uint32_t tmem, int* err) {
  tc_fence_before();
  __syncthreads();
  report_error(s.abort_flag, err);
  if (warp_id() == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Weights of four raw scores.  x: in, p out; m: what ds is multiplied by (p, or p tanh').  add: bias
// - lse in log2 units.  SMALL: see TanhSmall.
template <bool CAP, bool SMALL>
__device__ __forceinline__ void weights4(const Params& p, const TanhSmall& ts, float (&x)[4], const float (&add)[4],
                                         float (&m)[4]) {
  if (CAP) {
    cap4<SMALL>(p, ts, x, 0.f);
    const uint64_t inv = f2(p.cap_inv, p.cap_inv), neg = f2(-1.f, -1.f), one = f2(1.f, 1.f);
#pragma unroll
    for (int y = 0; y < 4; y += 2) {
      const uint64_t v = f2(x[y], x[y + 1]), t = f2_mul(v, inv);
      f2_split(f2_fma(f2_mul(t, neg), t, one), m[y], m[y + 1]);
      f2_split(f2_add(v, f2(add[y], add[y + 1])), x[y], x[y + 1]);
    }
  } else {
    const uint64_t c2 = f2(p.scale_log2, p.scale_log2);
    f2_split(f2_fma(f2(x[0], x[1]), c2, f2(add[0], add[1])), x[0], x[1]);
    f2_split(f2_fma(f2(x[2], x[3]), c2, f2(add[2], add[3])), x[2], x[3]);
  }
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    x[y] = ex2(x[y]);
    m[y] = CAP ? m[y] * x[y] : x[y];
  }
}

// fused_dkv.cu, fused_dq.cu
int launch_dkv(const BwdParams& f, const CUtensorMap& q, const CUtensorMap& go, const CUtensorMap& k,
               const CUtensorMap& v, int d, bool f16, bool cap, cudaStream_t s);
int launch_dq(const BwdParams& f, const CUtensorMap& q, const CUtensorMap& go, const CUtensorMap& k,
              const CUtensorMap& v, const CUtensorMap& dq, int d, bool f16, bool cap, cudaStream_t s);

}  // namespace fused
}  // namespace attn_bwd
