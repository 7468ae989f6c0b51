// fused_bwd.cuh — attention backward without materialised weights.
//
//   p = 2^(t - lse2)   dv = p^T do   dp = do v^T   ds = p (dp - delta) [tanh']   dq = scale ds k   dk = scale ds^T q
//
// Two kernels that each recompute p and dp, so that neither dq nor dk / dv needs atomics and
// equal inputs give equal bits; together 7 products of a tile pair instead of 5.
//   dkv: one key tile a CTA, streams the query tiles of all heads of the group.  It computes the
//        transposed scores (keys are rows), so p^T and ds^T are A operands in TMEM and the sum over
//        the group's heads happens in the accumulators.
//   dq:  one query tile of one head a CTA, streams the key tiles.
// In both, warp 8 is the TMA producer, warp 9 issues tcgen05, warp 10 fetches units (and makes their
// lists of tiles), and warps 0-7 turn scores into weights: TMEM lane quadrant warp % 4, columns
// 64 * (warp / 4).. of each tile.
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
  const float* nlse;     // [bs * H, sq_pad]: -lse * log2(e); -inf for rows that see nothing
  const float* ndelta;   // [bs * H, sq_pad]: -sum(do * o)
  void *dq, *dk, *dv;
  long long dqs[3], dks[3], dvs[3];   // element strides: batch, head, position
  float* part;           // dkv, splits > 1: [split][bs * Hkv * skv][2][D], dk first
};

template <int D>
struct BwdCfg {
  static constexpr int TILE_BYTES = TILE * D * 2;
  static constexpr int ST = 4;
  static constexpr int OFF_A = 0;                               // two resident tiles
  static constexpr int OFF_RING = 2 * TILE_BYTES;
  static constexpr int OFF_STAT = OFF_RING + ST * TILE_BYTES;   // dkv: 2 x (nlse, ndelta) of 128 rows
  static constexpr int OFF_STAGE = OFF_STAT + 2 * 2 * TILE * 4;
  static constexpr int OFF_LIST = OFF_STAGE + 8 * 2048;
  static constexpr int OFF_UNIT = OFF_LIST + 2 * kMaxList * 2;
  static constexpr int OFF_BAR = OFF_UNIT + 3 * 16;
  static constexpr int NBAR = 3 + 2 * ST + 6 + 6;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int SMEM_BYTES = OFF_MISC + 16 + 1024;
  static_assert(SMEM_BYTES <= 227 * 1024, "backward kernel shared memory");
};

struct BwdShared {
  uint8_t* smem;
  uint64_t *res_full, *res_empty, *all_done, *full, *empty, *s_full, *p_ready, *dp_full, *ds_ready, *done;
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
  s.dp_full = s.p_ready + 1;
  s.ds_ready = s.dp_full + 1;
  s.done = s.ds_ready + 1;
  s.sched.slot = reinterpret_cast<Unit*>(s.smem + C::OFF_UNIT);
  s.sched.handle = smem_u32(s.smem + C::OFF_UNIT + 32);
  s.sched.full = s.done + 1;
  s.sched.empty = s.sched.full + 2;
  s.sched.answer = s.sched.empty + 2;
  s.sched.ask = s.sched.answer + 1;
  s.tmem_slot = reinterpret_cast<uint32_t*>(s.smem + C::OFF_MISC);
  s.abort_flag = reinterpret_cast<volatile int*>(s.smem + C::OFF_MISC + 4);
  s.lists = reinterpret_cast<uint16_t*>(s.smem + C::OFF_LIST);
  return s;
}
// Barriers, descriptors and TMEM; returns the TMEM base.
__device__ __forceinline__ uint32_t bwd_begin(const BwdShared& s, int st, const CUtensorMap* q, const CUtensorMap* go,
                                              const CUtensorMap* k, const CUtensorMap* v) {
  const uint32_t warp = warp_id(), lane = lane_id();
  if (threadIdx.x == 0) {
    mbar_init(s.res_full, 1);
    mbar_init(s.res_empty, 1);
    mbar_init(s.all_done, 1);
    for (int i = 0; i < st; ++i) { mbar_init(&s.full[i], 1); mbar_init(&s.empty[i], 1); }
    mbar_init(&s.s_full[0], 1);
    mbar_init(&s.s_full[1], 1);
    mbar_init(s.p_ready, 8);
    mbar_init(s.dp_full, 1);
    mbar_init(s.ds_ready, 8);
    mbar_init(s.done, 1);
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

// nlse and ndelta of every row (rows of padding get -inf and 0).  16 lanes a row.
template <int D, bool F16>
__global__ void __launch_bounds__(256) bwd_stats_kernel(const uint8_t* __restrict__ go, const uint8_t* __restrict__ o,
                                                        const float* __restrict__ lse, float* __restrict__ nlse,
                                                        float* __restrict__ ndelta, int bs, int sq, int sq_pad, int H) {
  constexpr int L = D / 8;   // lanes a row: 16 bytes each
  const long long idx = ((long long)blockIdx.x * 256 + threadIdx.x) / L;   // (b, position, head)
  const int lane = threadIdx.x % L;
  const long long total = (long long)bs * sq_pad * H;
  const long long bp = idx / H, h = idx - bp * H, b = bp / sq_pad, pos = bp - b * sq_pad;
  const bool in = idx < total;
  float d = 0.f;
  if (in && pos < sq) {
    const long long at = ((b * sq + pos) * H + h) * (D * 2) + lane * 16;
    const uint4 x = *reinterpret_cast<const uint4*>(go + at), y = *reinterpret_cast<const uint4*>(o + at);
    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 u = unpack2<F16>(xs[i]), v = unpack2<F16>(ys[i]);
      d = fmaf(u.x, v.x, d);
      d = fmaf(u.y, v.y, d);
    }
  }
#pragma unroll
  for (int k = L / 2; k; k >>= 1) d += __shfl_xor_sync(0xffffffffu, d, k);
  if (in && lane == 0) {
    const float l = pos < sq ? lse[(b * H + h) * sq + pos] : -INFINITY;
    const bool none = l == -INFINITY;
    nlse[(b * H + h) * sq_pad + pos] = none ? -INFINITY : -l * kLog2e;
    ndelta[(b * H + h) * sq_pad + pos] = none ? 0.f : -d;
  }
}

// Weights of four scores.  x: raw scores in, p out; m: what ds is multiplied by (p, or p tanh').
// add: bias - lse in log2 units.
template <bool CAP>
__device__ __forceinline__ void weights4(const Params& p, float (&x)[4], const float (&add)[4], float (&m)[4]) {
  if (CAP) {
    float r[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) r[y] = x[y] * p.cap_in;
    cap_r4(r);
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      x[y] = fmaf(-2.f * p.cap_out, r[y], p.cap_out) + add[y];
      m[y] = 4.f * r[y] * (1.f - r[y]);
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
// ------------------------------------------------------------------------------- dk, dv
struct DkvUnit {
  int b, split, kvh, j0, j1, pre;
  int t_lo, nl;        // without documents: first visited query tile; tiles a head visits
  int i0, n;           // items of this unit: (head of the group, tile) pairs [i0, i0 + n)
};
__device__ __forceinline__ DkvUnit dkv_unit(const BwdParams& prm, const Unit& u) {
  const Params& p = prm.c;
  DkvUnit f;
  // earlier keys are seen by more queries and come first
  const int jt = prm.divHkv.div(u.x);
  f.kvh = u.x - jt * p.Hkv;
  f.b = u.y;
  f.split = u.z;
  f.j0 = jt * TILE;
  f.j1 = min(p.skv, f.j0 + TILE) - 1;
  f.pre = p.prefix ? __ldg(p.prefix + f.b) : 0;
  f.t_lo = 0;
  if (p.causal && f.j0 >= f.pre) f.t_lo = max(0, f.j0 - p.off) / TILE;   // rows from j0 - off on
  f.nl = p.has_docs ? u.n : max(0, p.n_tiles - f.t_lo);
  const int items = f.nl * p.G, per = (items + p.splits - 1) / p.splits;
  f.i0 = min(items, f.split * per);
  f.n = min(items, f.i0 + per) - f.i0;
  return f;
}
// Visited tile t (of nl): its number and flags.
__device__ __forceinline__ uint32_t dkv_entry(const Params& p, const DkvUnit& f, const uint16_t* list, int t, int& r0) {
  if (p.has_docs) {
    const uint32_t e = list[t];
    r0 = int(e & kEntTile) * TILE;
    return e;
  }
  r0 = (f.t_lo + t) * TILE;
  return row_limit(p, r0, f.pre) > f.j1 ? 0u : kEntMask;
}

template <int D, bool F16, bool CAP>
__global__ void __launch_bounds__(kThreads, 1)
dkv_kernel(const __grid_constant__ CUtensorMap tm_q,    // (d, s, h, b), box (64, 128, 1, 1)
           const __grid_constant__ CUtensorMap tm_do,   // the same
           const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const BwdParams prm) {
  using C = BwdCfg<D>;
  constexpr int ST = C::ST;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const BwdShared sh = bwd_shared<D>(smem_raw);
  const Params& p = prm.c;
  const uint32_t warp = warp_id(), lane = lane_id();
  const uint32_t tmem = bwd_begin(sh, ST, &tm_q, &tm_do, &tm_k, &tm_v);
  const uint32_t t_st = tmem, t_dp = tmem + TILE, t_dv = tmem + 2 * TILE, t_dk = t_dv + D;
  Unit u;

  if (warp >= 8) {
    regs_shrink();
    if (warp == 8) {
      // -------------------------------------------------------------- producer
      uint32_t it = 0, ri = 0;   // items and resident pairs loaded so far
      for (uint32_t k = 0; next_unit(sh.sched, k, u, sh.abort_flag, 0x3103); ++k) {
        const DkvUnit f = dkv_unit(prm, u);
        const uint16_t* list = sh.lists + (k & 1) * kMaxList;
        bool ok = true;
        if (f.n > 0) {
          ok = wait_for(sh.res_empty, (ri & 1) ^ 1, sh.abort_flag, 0x3102);
          if (!ok) break;
          ++ri;
          if (lane == 0) {
            mbar_arrive_expect_tx(sh.res_full, 2 * C::TILE_BYTES);
            for (int m = 0; m < 2; ++m)
              for (int x = 0; x < D / 64; ++x)
                tma_load_4d(sh.smem + C::OFF_A + m * C::TILE_BYTES + x * (TILE * 128), m ? &tm_v : &tm_k, sh.res_full,
                            x * 64, f.j0, f.kvh, f.b);
          }
          int g = f.i0 / f.nl, t = f.i0 - g * f.nl;
          for (int i = 0; i < f.n && ok; ++i, ++it) {
            int r0;
            dkv_entry(p, f, list, t, r0);
            const int h = f.kvh * p.G + g;
            for (int m = 0; m < 2; ++m) {
              const uint32_t s = (2 * it + m) % ST;
              ok = wait_for(&sh.empty[s], (((2 * it + m) / ST) & 1) ^ 1, sh.abort_flag, 0x3101);
              if (!ok) break;
              if (lane == 0) {
                mbar_arrive_expect_tx(&sh.full[s], C::TILE_BYTES + (m ? 0 : 2 * TILE * 4));
                for (int x = 0; x < D / 64; ++x)
                  tma_load_4d(sh.smem + C::OFF_RING + s * C::TILE_BYTES + x * (TILE * 128), m ? &tm_do : &tm_q,
                              &sh.full[s], x * 64, r0, h, f.b);
                if (!m) {   // the rows' statistics arrive with the queries
                  const size_t at = ((size_t)f.b * p.H + h) * prm.sq_pad + r0;
                  uint8_t* dst = sh.smem + C::OFF_STAT + (it & 1) * (2 * TILE * 4);
                  bulk_load(dst, prm.nlse + at, TILE * 4, &sh.full[s]);
                  bulk_load(dst + TILE * 4, prm.ndelta + at, TILE * 4, &sh.full[s]);
                }
              }
            }
            if (++t == f.nl) { t = 0; ++g; }
          }
        }
        if (!ok) break;
        ask_for_unit(sh.sched);
        unit_done(sh.sched, k);
      }
      if (lane == 0) {
        if (ri) mbar_drain(sh.res_full, (ri - 1) & 1, p.err, 0x3111);
        for (uint32_t k = 0; k < uint32_t(ST) && k < 2 * it; ++k) {
          const uint32_t i = 2 * it - 1 - k;
          mbar_drain(&sh.full[i % ST], (i / ST) & 1, p.err, 0x3112);
        }
      }
      __syncwarp();
    } else if (warp == 9) {
      // -------------------------------------------------------------- tensor cores
      constexpr uint32_t id_s = idesc16(F16, TILE, TILE, false, false);
      constexpr uint32_t id_g = idesc16(F16, TILE, D, false, true);
      const bool one = elect_one();
      const uint64_t ks = desc_k(smem_u32(sh.smem + C::OFF_A)), vs = desc_k(smem_u32(sh.smem + C::OFF_A) + C::TILE_BYTES);
      const uint32_t ring = smem_u32(sh.smem + C::OFF_RING);
      auto stage = [&](uint32_t si) { return ring + (si % ST) * C::TILE_BYTES; };
      uint32_t it = 0, ri = 0;
      bool ok = true;
      for (uint32_t k = 0; ok && next_unit(sh.sched, k, u, sh.abort_flag, 0x3208); ++k) {
        const DkvUnit f = dkv_unit(prm, u);
        const uint16_t* list = sh.lists + (k & 1) * kMaxList;
        if (f.n > 0) {
          // waits for slot si (and clears rows of padding: their products with 0 must be 0)
          auto arrived = [&](uint32_t si, int tt, int code) {
            if (!wait_for(&sh.full[si % ST], (si / ST) & 1, sh.abort_flag, code)) return false;
            if (p.has_docs && (list[tt] & kEntScrub)) {
              const int r0 = int(list[tt] & kEntTile) * TILE;
              scrub_rows<D>(stage(si), p.qdoc + (size_t)f.b * p.sq + r0, p.sq - r0, lane);
            }
            return true;
          };
          int t = f.i0 % f.nl;
          ok = wait_for(sh.res_full, ri & 1, sh.abort_flag, 0x3201) && arrived(2 * it, t, 0x3202) &&
               arrived(2 * it + 1, t, 0x3203);
          if (!ok) break;
          ++ri;
          tc_fence_after();
          mma_kk<D>(one, t_st, ks, desc_k(stage(2 * it)), id_s);
          commit1(one, &sh.s_full[0]);
          mma_kk<D>(one, t_dp, vs, desc_k(stage(2 * it + 1)), id_s);
          commit1(one, sh.dp_full);
          if (f.n == 1) commit1(one, sh.res_empty);
          for (int i = 0; i < f.n; ++i, ++it) {
            const bool more = i + 1 < f.n;
            if (++t == f.nl) t = 0;
            if (more && !(ok = arrived(2 * it + 2, t, 0x3204))) break;
            if (!(ok = wait_for(sh.p_ready, it & 1, sh.abort_flag, 0x3205))) break;
            tc_fence_after();
            mma_tn<D>(one, t_dv, t_st, t_st + 64, desc_mn(stage(2 * it + 1)), id_g, i > 0);
            commit1(one, &sh.empty[(2 * it + 1) % ST]);
            if (more) {
              mma_kk<D>(one, t_st, ks, desc_k(stage(2 * it + 2)), id_s);
              commit1(one, &sh.s_full[0]);
            }
            if (more && !(ok = arrived(2 * it + 3, t, 0x3206))) break;
            if (!(ok = wait_for(sh.ds_ready, it & 1, sh.abort_flag, 0x3207))) break;
            tc_fence_after();
            mma_tn<D>(one, t_dk, t_dp, t_dp + 64, desc_mn(stage(2 * it)), id_g, i > 0);
            commit1(one, &sh.empty[(2 * it) % ST]);
            if (more) {
              mma_kk<D>(one, t_dp, vs, desc_k(stage(2 * it + 3)), id_s);
              commit1(one, sh.dp_full);
              if (i + 2 == f.n) commit1(one, sh.res_empty);
            } else {
              commit1(one, sh.done);
            }
          }
          if (!ok) break;
        }
        unit_done(sh.sched, k);
      }
      // no commit may arrive after the block has left
      commit1(one, sh.all_done);
      wait_for(sh.all_done, 0, sh.abort_flag, 0x3209);
    } else if (warp == 10) {
      // -------------------------------------------------------------- units and their lists
      run_scheduler(sh.sched, sh.abort_flag, 0x3401, [&](int x, int y, int z, uint32_t slot) {
        if (!p.has_docs) return 0;
        const DkvUnit f = dkv_unit(prm, Unit{x, y, z, 0});
        const DocRange kd = prm.c.krange[(size_t)f.b * prm.n_kt + f.j0 / TILE];
        int n = 0;
        for (int t = f.t_lo; t < p.n_tiles; t += 32) {
          int st = kStSkip;
          bool scrub = false;
          if (t + int(lane) < p.n_tiles) {
            const int r0 = (t + int(lane)) * TILE;
            const DocRange qd = p.qrange[(size_t)f.b * p.n_tiles + t + lane];
            st = pair_state(p, f.pre, r0, min(p.sq, r0 + TILE) - 1, f.j0, f.j1, qd, kd);
            scrub = qd.neg != 0;
          }
          n = list_append(sh.lists + slot * kMaxList, n, t + int(lane), st, scrub, lane);
        }
        return n;
      });
    }
  } else {
    // ---------------------------------------------------------------- weights: one key a thread, 64 queries
    regs_grow();
    const int half = int(warp) >> 2;
    const uint32_t t_lane = uint32_t((warp & 3) * 32) << 16;
    const uint32_t st = t_st + t_lane + half * 64, dp = t_dp + t_lane + half * 64;
    const uint32_t stage = smem_u32(sh.smem + C::OFF_STAGE) + warp * 2048;
    const bool biased = p.slopes != nullptr;
    uint32_t it = 0, di = 0;
    bool ok = true;
    for (uint32_t k = 0; ok && next_unit(sh.sched, k, u, sh.abort_flag, 0x3305); ++k) {
      const DkvUnit f = dkv_unit(prm, u);
      const uint16_t* list = sh.lists + (k & 1) * kMaxList;
      const int j = f.j0 + int(warp & 3) * 32 + int(lane);
      const int kd = (p.has_docs && j < p.skv) ? __ldg(p.kdoc + (size_t)f.b * p.skv + j) : -1;
      int g = f.n > 0 ? f.i0 / f.nl : 0, t = f.n > 0 ? f.i0 - g * f.nl : 0;
      for (int i = 0; i < f.n; ++i, ++it) {
        int r0;
        const uint32_t ent = dkv_entry(p, f, list, t, r0);
        const bool masked = (ent & kEntMask) != 0;
        r0 += half * 64;   // first of this thread's query rows
        const float* stat = reinterpret_cast<const float*>(sh.smem + C::OFF_STAT + (it & 1) * (2 * TILE * 4)) + half * 64;
        uint32_t see[2] = {0xffffffffu, 0xffffffffu};
        if (masked) {
          // seen by row r if j < prefix or j <= r + off: rows from j - off on
          const int first = (!p.causal || j < f.pre) ? 0 : j - p.off - r0;
          if (p.has_docs) {
            int ids[2];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int r = r0 + y * 32 + int(lane);
              ids[y] = r < p.sq ? __ldg(p.qdoc + (size_t)f.b * p.sq + r) : -1;
            }
            same_ids<2>(ids, kd, see);
          }
#pragma unroll
          for (int y = 0; y < 2; ++y) see[y] &= ~low_bits(first - y * 32);
        }
        const float slope2 = biased ? __ldg(p.slopes + f.kvh * p.G + g) * kLog2e : 0.f;
        const float dist0 = float(r0 + p.off - j);
        ok = wait_for(&sh.s_full[0], it & 1, sh.abort_flag, 0x3301) &&
             wait_for(&sh.full[(2 * it) % ST], ((2 * it) / ST) & 1, sh.abort_flag, 0x3302);
        if (!ok) break;
        tc_fence_after();
        uint32_t w[2][32];   // scores, then what ds is multiplied by
#pragma unroll
        for (int y = 0; y < 2; ++y) tmem_ld32(st + y * 32, w[y]);
        tmem_wait_ld();
        auto phase = [&](auto bias_tag, auto mask_tag) {
          constexpr bool BIAS = decltype(bias_tag)::value, MASK = decltype(mask_tag)::value;
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 nl4 = *reinterpret_cast<const float4*>(stat + y * 32 + e);
              float add[4] = {nl4.x, nl4.y, nl4.z, nl4.w}, x[4], m[4];
#pragma unroll
              for (int z = 0; z < 4; ++z) {
                x[z] = __uint_as_float(w[y][e + z]);
                if (BIAS) add[z] = fmaf(-slope2, fabsf(dist0 + float(y * 32 + e + z)), add[z]);
              }
              weights4<CAP>(p, x, add, m);
#pragma unroll
              for (int z = 0; z < 4; ++z) {
                if (MASK && !((see[y] >> (e + z)) & 1u)) x[z] = m[z] = 0.f;
                w[y][e + z] = __float_as_uint(m[z]);
              }
              pk[e / 2] = pack2<F16>(x[0], x[1]);
              pk[e / 2 + 1] = pack2<F16>(x[2], x[3]);
            }
            tmem_st16(st + y * 16, pk);
          }
        };
        if (biased) {
          if (masked) phase(std::true_type{}, std::true_type{});
          else phase(std::true_type{}, std::false_type{});
        } else {
          if (masked) phase(std::false_type{}, std::true_type{});
          else phase(std::false_type{}, std::false_type{});
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(sh.p_ready);

        ok = wait_for(sh.dp_full, it & 1, sh.abort_flag, 0x3303);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          uint32_t d[32], pk[16];
          tmem_ld32(dp + y * 32, d);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 nd = *reinterpret_cast<const float4*>(stat + TILE + y * 32 + e);
            float a[4];
            f2_split(f2_mul(f2(w[y][e], w[y][e + 1]), f2_add(f2(d[e], d[e + 1]), f2(nd.x, nd.y))), a[0], a[1]);
            f2_split(f2_mul(f2(w[y][e + 2], w[y][e + 3]), f2_add(f2(d[e + 2], d[e + 3]), f2(nd.z, nd.w))), a[2], a[3]);
            if (masked) {   // p is 0 there already, but dp of padding may be NaN
#pragma unroll
              for (int z = 0; z < 4; ++z)
                if (!((see[y] >> (e + z)) & 1u)) a[z] = 0.f;
            }
            pk[e / 2] = pack2<F16>(a[0], a[1]);
            pk[e / 2 + 1] = pack2<F16>(a[2], a[3]);
          }
          tmem_st16(dp + y * 16, pk);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(sh.ds_ready);
        if (++t == f.nl) { t = 0; ++g; }
      }
      if (!ok) break;
      // ---- epilogue: warps 0-3 write dv, warps 4-7 dk
      if (f.n > 0) {
        ok = wait_for(sh.done, di & 1, sh.abort_flag, 0x3304);
        if (!ok) break;
        ++di;
      }
      tc_fence_after();
      const float fac = half ? p.scale : 1.f;
      const uint32_t src = (half ? t_dk : t_dv) + t_lane;
      uint8_t* out = half ? static_cast<uint8_t*>(prm.dk) + 2 * (f.b * prm.dks[0] + f.kvh * prm.dks[1] + j * prm.dks[2])
                          : static_cast<uint8_t*>(prm.dv) + 2 * (f.b * prm.dvs[0] + f.kvh * prm.dvs[1] + j * prm.dvs[2]);
      float* part = p.splits > 1
          ? prm.part + (((((size_t)f.split * p.bs + f.b) * p.Hkv + f.kvh) * p.skv + j) * 2 + (half ? 0 : 1)) * D : nullptr;
#pragma unroll 1
      for (int x = 0; x < D / 32; ++x) {
        uint32_t v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = 0u;
        __syncwarp();
        if (f.n > 0) {
          tmem_ld32(src + x * 32, v);
          tmem_wait_ld();
        }
        if (p.splits > 1) {
          if (j < p.skv) {
            float4* dst = reinterpret_cast<float4*>(part + x * 32);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              dst[e] = make_float4(__uint_as_float(v[4 * e]) * fac, __uint_as_float(v[4 * e + 1]) * fac,
                                   __uint_as_float(v[4 * e + 2]) * fac, __uint_as_float(v[4 * e + 3]) * fac);
          }
        } else {
          uint32_t o[16];
#pragma unroll
          for (int e = 0; e < 16; ++e)
            o[e] = pack2<F16>(__uint_as_float(v[2 * e]) * fac, __uint_as_float(v[2 * e + 1]) * fac);
          write_rows(stage, o, j < p.skv ? out + x * 64 : nullptr, lane);
        }
      }
      tc_fence_before();   // the next unit's first products overwrite the accumulators
      unit_done(sh.sched, k);
    }
  }
  bwd_end(sh, tmem, p.err);
}

// Sums the splits of dk and dv, in order.  D / 4 lanes a row of one of the two.
template <int D, bool F16>
__global__ void __launch_bounds__(256) dkv_join_kernel(const BwdParams prm) {
  const Params& p = prm.c;
  constexpr int L = D / 4;
  const long long idx = ((long long)blockIdx.x * 256 + threadIdx.x) / L;   // (b, kvh, j, which)
  const int lane = threadIdx.x % L;
  const long long rows = (long long)p.bs * p.Hkv * p.skv * 2;
  if (idx >= rows) return;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < p.splits; ++s) {
    const float4 x = *reinterpret_cast<const float4*>(prm.part + (s * rows + idx) * D + lane * 4);
    a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
  }
  const long long r = idx >> 1, bh = r / p.skv, j = r - bh * p.skv, b = bh / p.Hkv, h = bh - b * p.Hkv;
  uint8_t* out = (idx & 1) ? static_cast<uint8_t*>(prm.dv) + 2 * (b * prm.dvs[0] + h * prm.dvs[1] + j * prm.dvs[2])
                           : static_cast<uint8_t*>(prm.dk) + 2 * (b * prm.dks[0] + h * prm.dks[1] + j * prm.dks[2]);
  *reinterpret_cast<uint2*>(out + lane * 8) = make_uint2(pack2<F16>(a.x, a.y), pack2<F16>(a.z, a.w));
}

// ------------------------------------------------------------------------------- dq
struct DqUnit {
  int b, h, kvh, r0, r1, pre, lim0, n;
};
__device__ __forceinline__ DqUnit dq_unit(const BwdParams& prm, const Unit& u) {
  const Params& p = prm.c;
  DqUnit f;
  const int blk = prm.divH.div(u.x), qt = p.n_tiles - 1 - blk;   // later queries see more: first
  f.h = u.x - blk * p.H;
  f.b = u.y;
  f.kvh = p.divG.div(f.h);
  f.r0 = qt * TILE;
  f.r1 = min(p.sq, f.r0 + TILE) - 1;
  f.pre = p.prefix ? __ldg(p.prefix + f.b) : 0;
  f.lim0 = row_limit(p, f.r0, f.pre);
  f.n = p.has_docs ? u.n : max(0, row_limit(p, f.r1, f.pre) + TILE - 1) / TILE;
  return f;
}

// TMEM: two score tiles (the next one is computed while this one is worked on; ds is written
// over the scores it came from), dp, and the accumulator.
template <int D, bool F16, bool CAP>
__global__ void __launch_bounds__(kThreads, 1)
dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
          const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const BwdParams prm) {
  using C = BwdCfg<D>;
  constexpr int ST = C::ST;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const BwdShared sh = bwd_shared<D>(smem_raw);
  const Params& p = prm.c;
  const uint32_t warp = warp_id(), lane = lane_id();
  const uint32_t tmem = bwd_begin(sh, ST, &tm_q, &tm_do, &tm_k, &tm_v);
  const uint32_t t_dp = tmem + 2 * TILE, t_dq = tmem + 3 * TILE;
  Unit u;

  if (warp >= 8) {
    regs_shrink();
    if (warp == 8) {
      // -------------------------------------------------------------- producer
      uint32_t it = 0, ri = 0;
      for (uint32_t k = 0; next_unit(sh.sched, k, u, sh.abort_flag, 0x4103); ++k) {
        const DqUnit f = dq_unit(prm, u);
        const uint16_t* list = sh.lists + (k & 1) * kMaxList;
        bool ok = true;
        if (f.n > 0) {
          ok = wait_for(sh.res_empty, (ri & 1) ^ 1, sh.abort_flag, 0x4102);
          if (!ok) break;
          ++ri;
          if (lane == 0) {
            mbar_arrive_expect_tx(sh.res_full, 2 * C::TILE_BYTES);
            for (int m = 0; m < 2; ++m)
              for (int x = 0; x < D / 64; ++x)
                tma_load_4d(sh.smem + C::OFF_A + m * C::TILE_BYTES + x * (TILE * 128), m ? &tm_do : &tm_q, sh.res_full,
                            x * 64, f.r0, f.h, f.b);
          }
        }
        for (int i = 0; i < f.n && ok; ++i, ++it) {
          const int j0 = (p.has_docs ? int(list[i] & kEntTile) : i) * TILE;
          for (int m = 0; m < 2; ++m) {
            const uint32_t s = (2 * it + m) % ST;
            ok = wait_for(&sh.empty[s], (((2 * it + m) / ST) & 1) ^ 1, sh.abort_flag, 0x4101);
            if (!ok) break;
            if (lane == 0) {
              mbar_arrive_expect_tx(&sh.full[s], C::TILE_BYTES);
              for (int x = 0; x < D / 64; ++x)
                tma_load_4d(sh.smem + C::OFF_RING + s * C::TILE_BYTES + x * (TILE * 128), m ? &tm_v : &tm_k,
                            &sh.full[s], x * 64, j0, f.kvh, f.b);
            }
          }
        }
        if (!ok) break;
        ask_for_unit(sh.sched);
        unit_done(sh.sched, k);
      }
      if (lane == 0) {
        if (ri) mbar_drain(sh.res_full, (ri - 1) & 1, p.err, 0x4111);
        for (uint32_t k = 0; k < uint32_t(ST) && k < 2 * it; ++k) {
          const uint32_t i = 2 * it - 1 - k;
          mbar_drain(&sh.full[i % ST], (i / ST) & 1, p.err, 0x4112);
        }
      }
      __syncwarp();
    } else if (warp == 9) {
      // -------------------------------------------------------------- tensor cores
      constexpr uint32_t id_s = idesc16(F16, TILE, TILE, false, false);
      constexpr uint32_t id_g = idesc16(F16, TILE, D, false, true);
      const bool one = elect_one();
      const uint64_t qs = desc_k(smem_u32(sh.smem + C::OFF_A)), dos = desc_k(smem_u32(sh.smem + C::OFF_A) + C::TILE_BYTES);
      const uint32_t ring = smem_u32(sh.smem + C::OFF_RING);
      auto stage = [&](uint32_t si) { return ring + (si % ST) * C::TILE_BYTES; };
      uint32_t it = 0, ri = 0;
      bool ok = true;
      for (uint32_t k = 0; ok && next_unit(sh.sched, k, u, sh.abort_flag, 0x4208); ++k) {
        const DqUnit f = dq_unit(prm, u);
        const uint16_t* list = sh.lists + (k & 1) * kMaxList;
        if (f.n > 0) {
          auto arrived = [&](int i, int m, int code) {   // key (m = 0) or value tile of the unit's item i
            const uint32_t si = 2 * (it + i) + m;
            if (!wait_for(&sh.full[si % ST], (si / ST) & 1, sh.abort_flag, code)) return false;
            return true;
          };
          auto scrub = [&](int i, uint32_t si) {
            if (p.has_docs && (list[i] & kEntScrub)) {
              const int j0 = int(list[i] & kEntTile) * TILE;
              scrub_rows<D>(stage(si), p.kdoc + (size_t)f.b * p.skv + j0, p.skv - j0, lane);
            }
          };
          ok = wait_for(sh.res_full, ri & 1, sh.abort_flag, 0x4201) && arrived(0, 0, 0x4202) &&
               arrived(0, 1, 0x4203) && (f.n < 2 || arrived(1, 0, 0x4204));
          if (!ok) break;
          ++ri;
          scrub(0, 2 * it);
          if (f.n > 1) scrub(1, 2 * it + 2);
          tc_fence_after();
          mma_kk<D>(one, tmem + (it & 1) * TILE, qs, desc_k(stage(2 * it)), id_s);
          commit1(one, &sh.s_full[it & 1]);
          mma_kk<D>(one, t_dp, dos, desc_k(stage(2 * it + 1)), id_s);
          commit1(one, sh.dp_full);
          commit1(one, &sh.empty[(2 * it + 1) % ST]);
          if (f.n > 1) {
            mma_kk<D>(one, tmem + ((it + 1) & 1) * TILE, qs, desc_k(stage(2 * it + 2)), id_s);
            commit1(one, &sh.s_full[(it + 1) & 1]);
          } else {
            commit1(one, sh.res_empty);
          }
          for (int i = 0; i < f.n; ++i, ++it) {
            if (i + 1 < f.n && !(ok = arrived(1, 1, 0x4205))) break;
            if (!(ok = wait_for(sh.ds_ready, it & 1, sh.abort_flag, 0x4206))) break;
            tc_fence_after();
            const uint32_t t_s = tmem + (it & 1) * TILE;
            if (i + 1 < f.n) {
              mma_kk<D>(one, t_dp, dos, desc_k(stage(2 * it + 3)), id_s);
              commit1(one, sh.dp_full);
              commit1(one, &sh.empty[(2 * it + 3) % ST]);
              if (i + 2 == f.n) commit1(one, sh.res_empty);   // the last scores were issued before
            }
            mma_tn<D>(one, t_dq, t_s, t_s + 64, desc_mn(stage(2 * it)), id_g, i > 0);
            commit1(one, &sh.empty[(2 * it) % ST]);
            if (i + 1 == f.n) commit1(one, sh.done);
            if (i + 2 < f.n) {
              if (!(ok = arrived(2, 0, 0x4207))) break;
              scrub(i + 2, 2 * it + 4);
              tc_fence_after();
              mma_kk<D>(one, t_s, qs, desc_k(stage(2 * it + 4)), id_s);
              commit1(one, &sh.s_full[it & 1]);
            }
          }
          if (!ok) break;
        }
        unit_done(sh.sched, k);
      }
      // no commit may arrive after the block has left
      commit1(one, sh.all_done);
      wait_for(sh.all_done, 0, sh.abort_flag, 0x4209);
    } else if (warp == 10) {
      // -------------------------------------------------------------- units and their lists
      run_scheduler(sh.sched, sh.abort_flag, 0x4401, [&](int x, int y, int z, uint32_t slot) {
        if (!p.has_docs) return 0;
        const DqUnit f = dq_unit(prm, Unit{x, y, z, 0});
        const DocRange qd = p.qrange[(size_t)f.b * p.n_tiles + f.r0 / TILE];
        const int t1 = max(0, row_limit(p, f.r1, f.pre) + TILE - 1) / TILE;
        int n = 0;
        for (int t = 0; t < t1; t += 32) {
          int st = kStSkip;
          bool scrub = false;
          if (t + int(lane) < t1) {
            const int j0 = (t + int(lane)) * TILE;
            const DocRange kd = p.krange[(size_t)f.b * prm.n_kt + t + lane];
            st = pair_state(p, f.pre, f.r0, f.r1, j0, j0 + TILE - 1, qd, kd);
            scrub = kd.neg != 0;
          }
          n = list_append(sh.lists + slot * kMaxList, n, t + int(lane), st, scrub, lane);
        }
        return n;
      });
    }
  } else {
    // ---------------------------------------------------------------- weights: one query a thread, 64 keys
    regs_grow();
    const int half = int(warp) >> 2;
    const uint32_t t_lane = uint32_t((warp & 3) * 32) << 16;
    const uint32_t dp = t_dp + t_lane + half * 64;
    const uint32_t stage = smem_u32(sh.smem + C::OFF_STAGE) + warp * 2048;
    const bool biased = p.slopes != nullptr;
    uint32_t it = 0, di = 0;
    bool ok = true;
    for (uint32_t k = 0; ok && next_unit(sh.sched, k, u, sh.abort_flag, 0x4304); ++k) {
      const DqUnit f = dq_unit(prm, u);
      const uint16_t* list = sh.lists + (k & 1) * kMaxList;
      const int row = f.r0 + int(warp & 3) * 32 + int(lane);
      const bool valid = row < p.sq;
      const size_t ri = ((size_t)f.b * p.H + f.h) * prm.sq_pad + row;
      const float nlse = prm.nlse[ri], nd = prm.ndelta[ri];   // padded to whole tiles
      const int lim = valid ? row_limit(p, row, f.pre) : 0;
      const int qd = (valid && p.has_docs) ? __ldg(p.qdoc + (size_t)f.b * p.sq + row) : -1;
      const float slope2 = biased ? __ldg(p.slopes + f.h) * kLog2e : 0.f;
      const uint64_t nd2 = f2(nd, nd);
      for (int i = 0; i < f.n; ++i, ++it) {
        const uint32_t ent = p.has_docs ? list[i] : 0u;
        const int t0 = (p.has_docs ? int(ent & kEntTile) : i) * TILE, j0 = t0 + half * 64;
        const bool masked = p.has_docs ? (ent & kEntMask) != 0 : t0 + TILE > f.lim0;
        const uint32_t st = tmem + (it & 1) * TILE + t_lane + half * 64;
        uint32_t see[2] = {0xffffffffu, 0xffffffffu};
        if (masked) {
          if (p.has_docs) {
            int ids[2];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int j = j0 + y * 32 + int(lane);
              ids[y] = j < p.skv ? __ldg(p.kdoc + (size_t)f.b * p.skv + j) : -1;
            }
            same_ids<2>(ids, qd, see);
          }
#pragma unroll
          for (int y = 0; y < 2; ++y) see[y] &= low_bits(lim - j0 - y * 32);
        }
        ok = wait_for(&sh.s_full[it & 1], (it >> 1) & 1, sh.abort_flag, 0x4301);
        if (!ok) break;
        tc_fence_after();
        uint32_t w[2][32];
#pragma unroll
        for (int y = 0; y < 2; ++y) tmem_ld32(st + y * 32, w[y]);
        tmem_wait_ld();
        const float dist0 = float(row + p.off - j0);
        auto phase = [&](auto bias_tag) {
          constexpr bool BIAS = decltype(bias_tag)::value;
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              float add[4], x[4], m[4];
#pragma unroll
              for (int z = 0; z < 4; ++z) {
                x[z] = __uint_as_float(w[y][e + z]);
                add[z] = BIAS ? fmaf(-slope2, fabsf(dist0 - float(y * 32 + e + z)), nlse) : nlse;
              }
              weights4<CAP>(p, x, add, m);
#pragma unroll
              for (int z = 0; z < 4; ++z) w[y][e + z] = __float_as_uint(m[z]);
            }
        };
        // masked scores are taken out of ds below
        if (biased) phase(std::true_type{});
        else phase(std::false_type{});
        ok = wait_for(sh.dp_full, it & 1, sh.abort_flag, 0x4302);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          uint32_t d[32], pk[16];
          tmem_ld32(dp + y * 32, d);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float a0, a1;
            f2_split(f2_mul(f2(w[y][e], w[y][e + 1]), f2_add(f2(d[e], d[e + 1]), nd2)), a0, a1);
            if (masked) {
              if (!((see[y] >> e) & 1u)) a0 = 0.f;
              if (!((see[y] >> (e + 1)) & 1u)) a1 = 0.f;
            }
            pk[e / 2] = pack2<F16>(a0, a1);
          }
          tmem_st16(st + y * 16, pk);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(sh.ds_ready);
      }
      if (!ok) break;
      // ---- epilogue: each half of the warps writes half of the columns
      if (f.n > 0) {
        ok = wait_for(sh.done, di & 1, sh.abort_flag, 0x4303);
        if (!ok) break;
        ++di;
      }
      tc_fence_after();
      uint8_t* out = static_cast<uint8_t*>(prm.dq) + 2 * (f.b * prm.dqs[0] + f.h * prm.dqs[1] + row * prm.dqs[2]) +
                     half * D;
#pragma unroll 1
      for (int x = 0; x < D / 64; ++x) {
        uint32_t v[32], o[16];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = 0u;
        __syncwarp();
        if (f.n > 0) {
          tmem_ld32(t_dq + t_lane + half * (D / 2) + x * 32, v);
          tmem_wait_ld();
        }
#pragma unroll
        for (int e = 0; e < 16; ++e)
          o[e] = pack2<F16>(__uint_as_float(v[2 * e]) * p.scale, __uint_as_float(v[2 * e + 1]) * p.scale);
        write_rows(stage, o, valid ? out + x * 64 : nullptr, lane);
      }
      tc_fence_before();   // the next unit's first product overwrites the accumulator
      unit_done(sh.sched, k);
    }
  }
  bwd_end(sh, tmem, p.err);
}

}  // namespace fused
}  // namespace attn_bwd
