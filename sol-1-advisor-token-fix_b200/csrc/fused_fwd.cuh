// fused_fwd.cuh — attention forward: o = softmax(modified scores) v, with the row statistic
// lse = log(sum(exp(s))), in one pass over the keys (running maximum and sum).
//
// One CTA holds up to two query tiles of 128 rows and streams key / value tiles of 128 keys
// through a ring in shared memory; both tiles use each of them.  While the tensor cores work
// for one query tile, the other one's softmax runs:
//   warp 8  TMA producer      warp 9  tcgen05 issuer, TMEM owner      warp 10  units and their lists
//   warps 0-3 softmax of tile 0, warps 4-7 of tile 1: one thread a row
// A CTA stays on its SM and takes up unit after unit: the next unit's tiles are loaded and its
// first scores computed while this one's rows are still written.
// TMEM: two score tiles (128 columns each) and two outputs (D columns each).  The weights go
// back to TMEM as 16-bit pairs over the scores they came from and are the A operand of the
// second product, so they never touch shared memory.  They are handed over in two halves, so
// the second product starts while the second half is still computed.
//
// The running maximum lags: the accumulator is rescaled only where a row's maximum has grown by
// more than 2^8, so most tiles need no pass over it.  Weights are then at most 2^8 instead of
// 1, which neither fp32 sums nor 16-bit weights (relative rounding) notice.
//
// Where all rows of a unit fit one tile (generated tokens), the two sets of warps take alternate key
// tiles for the same rows instead (DUO): what bounds such a unit is the chain of scores, softmax and
// product per tile, and two chains run side by side.  Each leaves its part to be joined.
//
// What bounds it: with few rows the keys and values, read once (4 tokens over 8191 keys, 80 + 8 heads of
// 128: 28 us, 4.8 TB/s); with many, turning scores into weights: 4096 x 4096, 80 + 8 heads of 128, bf16
// take 557 us without a mask (1.23 PFLOP/s) and 298 us causal (1.15 of what is seen), where the
// tensor cores are active half of the time and the exponentials' unit as long.  A bias costs 453
// us, a cap 432 (both causal), since each adds instructions to every score.  (These are bursts on a
// cool GPU.  Back to back for longer, the power limit lowers the clock: 608 us without a mask, 345 causal.)
//
// Rows of a query tile are 128 positions of one head or, where that needs fewer tiles, up to
// 128 (position, head) pairs of one group (few positions, as when tokens are generated): a
// group's heads read the same keys.
#pragma once
#include <type_traits>

#include "fused_common.cuh"
#include "fused_host.h"

namespace attn_bwd {
namespace fused {

struct FwdParams {
  Params c;
  int cta_splits;      // splits of the grid; DUO leaves two parts each
  int packed;          // rows are (position, head of the group) pairs
  int pos_per_tile;    // positions of a tile: 128, or 128 / G
  int duo;             // all rows of a unit in one tile: two chains over alternate key tiles
  int pair_heads;      // unpacked: the two tiles are two heads of one group, else 256 positions
  int blocks_q;        // position blocks per (batch, head slot)
  int wide;            // rows of o start at multiples of 32 bytes
  int head_slots;      // units along the heads: kv heads, head pairs or heads
  FastDiv div_slots;
  void* o;             // [bs, sq, H, D]
  float* lse;          // [bs, H, sq]
  float* part_o;       // splits > 1: [split][bs * H * sq][D]
  float* part_lse;     // splits > 1: [split][bs * H * sq]
};

template <int D, bool DUO>
struct FwdCfg {
  static constexpr int TILE_BYTES = TILE * D * 2;
  static constexpr int QT = DUO ? 1 : 2;                       // query tiles
  static constexpr int ST = (D == 128 ? 6 : 10) - QT;          // stages of keys or values
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_KV = QT * TILE_BYTES;
  static constexpr int OFF_STAGE = OFF_KV + ST * TILE_BYTES;   // 2 KB for each warp of rows
  static constexpr int OFF_LIST = OFF_STAGE + (DUO ? 0 : 8 * 2048);   // a list for each unit slot
  static constexpr int OFF_UNIT = OFF_LIST + 2 * kMaxList * 2;
  static constexpr int OFF_BAR = OFF_UNIT + 3 * 16;            // two slots, the scheduler's answer
  static constexpr int NBAR = 3 + 2 * ST + 8 + 6;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int SMEM_BYTES = OFF_MISC + 16 + 1024;
  static_assert(SMEM_BYTES <= 227 * 1024, "forward kernel shared memory");
};

// What a unit is: its tiles' heads and positions, and the key tiles it visits.
struct FwdUnit {
  int b, split, kvh, nt;
  int head[2], pos[2];
  int last_pos;
  int t0, n;          // first key tile of the split, number of visited ones
  int pre, lim0;      // prefix; number of keys that the first row sees (documents aside)
};
__device__ __forceinline__ FwdUnit fwd_unit(const FwdParams& prm, const Unit& u) {
  const Params& p = prm.c;
  FwdUnit f;
  // later positions see more keys and come first
  const int blk = prm.div_slots.div(u.x);
  const int qb = prm.blocks_q - 1 - blk;
  const int slot = u.x - blk * prm.head_slots;
  f.b = u.y;
  f.split = u.z;
  if (prm.packed) {
    f.kvh = slot;
    f.head[0] = f.head[1] = slot * p.G;
    f.pos[0] = qb * 2 * prm.pos_per_tile;
    f.pos[1] = f.pos[0] + prm.pos_per_tile;
  } else if (prm.pair_heads) {
    f.head[0] = slot * 2;
    f.head[1] = slot * 2 + 1;
    f.kvh = p.divG.div(f.head[0]);
    f.pos[0] = f.pos[1] = qb * TILE;
  } else {
    f.head[0] = f.head[1] = slot;
    f.kvh = p.divG.div(slot);
    f.pos[0] = qb * 2 * TILE;
    f.pos[1] = f.pos[0] + TILE;
  }
  f.nt = f.pos[1] < p.sq ? 2 : 1;
  f.last_pos = min(p.sq, (f.nt == 2 ? f.pos[1] : f.pos[0]) + prm.pos_per_tile) - 1;
  f.pre = p.prefix ? __ldg(p.prefix + f.b) : 0;
  f.lim0 = row_limit(p, f.pos[0], f.pre);
  f.t0 = f.split * p.tiles_per_split;
  const int hi = max(0, row_limit(p, f.last_pos, f.pre) + TILE - 1) / TILE;
  f.n = p.has_docs ? u.n : max(0, min(min(p.n_tiles, f.t0 + p.tiles_per_split), hi) - f.t0);
  return f;
}
template <int D, bool F16, bool CAP, bool BIAS, bool DUO>
__global__ void __launch_bounds__(kThreads, 1)
fwd_kernel(const __grid_constant__ CUtensorMap tm_q,   // (d, h, s, b), box (64, heads of a row, positions, 1)
           const __grid_constant__ CUtensorMap tm_k,   // (d, s, h, b), box (64, 128, 1, 1)
           const __grid_constant__ CUtensorMap tm_v,
           const __grid_constant__ CUtensorMap tm_o,   // (d, h, s, b), box (32, 1, 32, 1): unpacked rows' results
           const FwdParams prm) {
  using C = FwdCfg<D, DUO>;
  constexpr int ST = C::ST;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* all_done = bars + 2;
  uint64_t* kv_full = bars + 3;
  uint64_t* kv_empty = kv_full + ST;
  uint64_t* s_full = kv_empty + ST;    // [tile] scores ready
  uint64_t* p_ready = s_full + 2;      // [tile][half] weights written
  uint64_t* o_done = p_ready + 4;      // [tile] second product done
  Scheduler sched;
  sched.slot = reinterpret_cast<Unit*>(smem + C::OFF_UNIT);
  sched.handle = smem_u32(smem + C::OFF_UNIT + 32);
  sched.full = o_done + 2;
  sched.empty = sched.full + 2;
  sched.answer = sched.empty + 2;
  sched.ask = sched.answer + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 4);
  uint16_t* lists = reinterpret_cast<uint16_t*>(smem + C::OFF_LIST);

  const Params& p = prm.c;
  const uint32_t warp = warp_id(), lane = lane_id();
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(all_done, 1);
    for (int i = 0; i < ST; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 1); }
    for (int i = 0; i < 4; ++i) mbar_init(&p_ready[i], 4);
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&o_done[i], 1); }
    scheduler_init(sched);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 8 && lane == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  if (warp == 9) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  wait_for_previous();
  if (prm.packed) {
    // rows behind the last (position, head) pair of a tile are never loaded; what stood there
    // would take part in the warps' votes, and results would not be the same bits each time
    const int r0 = prm.pos_per_tile * p.G, n = (TILE - r0) * (D / 8);
    for (int i = int(threadIdx.x); i < C::QT * n; i += kThreads) {
      const int t = i >= n ? 1 : 0, j = i - t * n, c = j % (D / 8), r = r0 + j / (D / 8);
      sts128(smem_u32(smem + C::OFF_Q + t * C::TILE_BYTES + (c >> 3) * (TILE * 128)) + r * 128 + (c & 7) * 16,
             make_uint4(0, 0, 0, 0));
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Unit u;

  if (warp >= 8) {
    regs_shrink();
    if (warp == 8) {
      // -------------------------------------------------------------- producer
      uint32_t si = 0, qi = 0, round = 0;   // key / value tiles, query tiles loaded so far; DUO: rounds
      for (uint32_t k = 0; next_unit(sched, k, u, abort_flag, 0x2103); ++k) {
        const FwdUnit f = fwd_unit(prm, u);
        const uint16_t* list = lists + (k & 1) * kMaxList;
        bool ok = true;
        if (f.n > 0) {
          ok = wait_for(q_empty, (qi & 1) ^ 1, abort_flag, 0x2102);
          if (!ok) break;
          ++qi;
          if (lane == 0) {
            // a tile's box covers pos_per_tile positions x 1 head, or x the group's heads
            const int rows = prm.packed ? prm.pos_per_tile * p.G : TILE;
            mbar_arrive_expect_tx(q_full, uint32_t(f.nt) * rows * D * 2);
            for (int t = 0; t < f.nt; ++t)
              for (int x = 0; x < D / 64; ++x)
                tma_load_4d(smem + C::OFF_Q + t * C::TILE_BYTES + x * (TILE * 128), &tm_q, q_full, x * 64,
                            t ? f.head[1] : f.head[0], t ? f.pos[1] : f.pos[0], f.b);
          }
        }
        // a key (m = 0) or value tile into the stage of ring index r
        auto load = [&](uint32_t r, int i, int m) {
          const int j0 = (f.t0 + (p.has_docs ? int(list[i] & kEntTile) : i)) * TILE;
          const uint32_t s = r % ST;
          if (!wait_for(&kv_empty[s], ((r / ST) & 1) ^ 1, abort_flag, 0x2101)) return false;
          if (lane == 0) {
            mbar_arrive_expect_tx(&kv_full[s], C::TILE_BYTES);
            for (int x = 0; x < D / 64; ++x)
              tma_load_4d(smem + C::OFF_KV + s * C::TILE_BYTES + x * (TILE * 128), m ? &tm_v : &tm_k, &kv_full[s],
                          x * 64, j0, f.kvh, f.b);
          }
          return true;
        };
        auto pass = [&](uint32_t r) {
          if (!wait_for(&kv_empty[r % ST], ((r / ST) & 1) ^ 1, abort_flag, 0x2104)) return false;
          if (lane == 0) mbar_arrive(&kv_full[r % ST]);
          return true;
        };
        if (DUO) {
          // rounds of four stages: keys of both chains, values of both; after a last odd tile two
          // stages of its round are passed on as they are
          for (int i = 0; i < f.n && ok; i += 2, ++round) {
            const bool two = i + 1 < f.n;
            ok = load(4 * round, i, 0) && (!two || load(4 * round + 1, i + 1, 0)) && load(4 * round + 2, i, 1) &&
                 (!two || load(4 * round + 3, i + 1, 1));
            if (ok && !two) ok = pass(4 * round + 1) && pass(4 * round + 3);
          }
        } else {
          for (int i = 0; i < f.n && ok; ++i, si += 2) ok = load(si, i, 0) && load(si + 1, i, 1);
        }
        if (!ok) break;
        ask_for_unit(sched);
        unit_done(sched, k);
      }
      if (DUO) si = 4 * round;
      if (lane == 0) {
        if (qi) mbar_drain(q_full, (qi - 1) & 1, p.err, 0x2111);
        for (uint32_t k = 0; k < uint32_t(ST) && k < si; ++k) {
          const uint32_t i = si - 1 - k;
          mbar_drain(&kv_full[i % ST], (i / ST) & 1, p.err, 0x2112);
        }
      }
      __syncwarp();
    } else if (warp == 9) {
      // -------------------------------------------------------------- tensor cores
      const bool one = elect_one();
      constexpr uint32_t id_s = idesc16(F16, TILE, TILE, false, false);
      constexpr uint32_t id_o = idesc16(F16, TILE, D, false, true);
      const uint32_t qs = smem_u32(smem + C::OFF_Q), kvs = smem_u32(smem + C::OFF_KV);
      auto stage = [&](uint32_t si) { return kvs + (si % ST) * C::TILE_BYTES; };
      auto full = [&](uint32_t si, int code) {
        return wait_for(&kv_full[si % ST], (si / ST) & 1, abort_flag, code);
      };
      uint32_t si = 0, qi = 0, cnt[2] = {0, 0};
      for (uint32_t k = 0; next_unit(sched, k, u, abort_flag, 0x2200); ++k) {
        const FwdUnit f = fwd_unit(prm, u);
        const uint16_t* list = lists + (k & 1) * kMaxList;
        // clears the padding of a key or value tile (the unit's i-th, ring index r).  Values: a NaN there times
        // a weight of 0 is NaN.  Keys: only below a cap, where four scores share a reciprocal and a warp
        // its choice of the tanh's form; their scores are hidden after it.
        auto scrub = [&](uint32_t r, int i) {
          if (p.has_docs && (list[i] & kEntScrub)) {
            const int j0 = (f.t0 + int(list[i] & kEntTile)) * TILE;
            scrub_rows<D>(stage(r), p.kdoc + (size_t)f.b * p.skv + j0, p.skv - j0, lane);
          }
        };
        if (DUO && f.n > 0) {
          if (!wait_for(q_full, qi & 1, abort_flag, 0x2201)) break;
          ++qi;
          // scores of tile j (ring index r of its keys), or a stage passed on
          auto scores = [&](uint32_t r, int j) {
            if (!full(r, 0x2202)) return false;
            if (j < f.n) {
              if (CAP) scrub(r, j);
              tc_fence_after();
              mma_kk<D>(one, tmem + (j & 1) * TILE, desc_k(qs), desc_k(stage(r)), id_s);
              commit1(one, &s_full[j & 1]);
            }
            commit1(one, &kv_empty[r % ST]);
            return true;
          };
          bool ok = scores(si, 0) && scores(si + 1, 1);
          for (int i = 0; i < f.n && ok; i += 2, si += 4)
            for (int t = 0; t < 2 && ok; ++t) {
              const int j = i + t;
              const uint32_t r = si + 2 + t;
              if (!(ok = full(r, 0x2203))) break;
              if (j < f.n) {
                scrub(r, j);
                const uint32_t t_s = tmem + t * TILE, t_o = tmem + 2 * TILE + t * D;
                if (!(ok = wait_for(&p_ready[2 * t], cnt[t] & 1, abort_flag, 0x2205))) break;
                tc_fence_after();
                mma_tn<D, 0, 4>(one, t_o, t_s, t_s + 32, desc_mn(stage(r)), id_o, i > 0);
                if (!(ok = wait_for(&p_ready[2 * t + 1], cnt[t] & 1, abort_flag, 0x2206))) break;
                tc_fence_after();
                mma_tn<D, 4, 8>(one, t_o, t_s, t_s + 32, desc_mn(stage(r)), id_o, true);
                commit1(one, &o_done[t]);
                ++cnt[t];
              }
              commit1(one, &kv_empty[r % ST]);
              if (i + 2 < f.n) ok = scores(si + 4 + t, j + 2);
            }
          if (!ok) break;
          commit1(one, q_empty);
        }
        if (!DUO && f.n > 0) {
          if (!wait_for(q_full, qi & 1, abort_flag, 0x2201) || !full(si, 0x2202)) break;
          ++qi;
          if (CAP) scrub(si, 0);
          tc_fence_after();
          for (int t = 0; t < f.nt; ++t) {
            mma_kk<D>(one, tmem + t * TILE, desc_k(qs + t * C::TILE_BYTES), desc_k(stage(si)), id_s);
            commit1(one, &s_full[t]);
          }
          commit1(one, &kv_empty[si % ST]);
          if (f.n == 1) commit1(one, q_empty);
          bool ok = true;
          for (int i = 0; i < f.n; ++i) {
            const uint32_t vi = si + 1, kn = si + 2;
            const bool more = i + 1 < f.n;
            if (!(ok = full(vi, 0x2203))) break;
            scrub(vi, i);
            if (more && !(ok = full(kn, 0x2204))) break;
            if (CAP && more) scrub(kn, i + 1);
            for (int t = 0; t < f.nt && ok; ++t) {
              const uint32_t t_s = tmem + t * TILE, t_o = tmem + 2 * TILE + t * D;
              ok = wait_for(&p_ready[2 * t], (cnt[t] + i) & 1, abort_flag, 0x2205);
              if (!ok) break;
              tc_fence_after();
              mma_tn<D, 0, 4>(one, t_o, t_s, t_s + 32, desc_mn(stage(vi)), id_o, i > 0);
              ok = wait_for(&p_ready[2 * t + 1], (cnt[t] + i) & 1, abort_flag, 0x2206);
              if (!ok) break;
              tc_fence_after();
              mma_tn<D, 4, 8>(one, t_o, t_s, t_s + 32, desc_mn(stage(vi)), id_o, true);
              commit1(one, &o_done[t]);
              if (t == f.nt - 1) commit1(one, &kv_empty[vi % ST]);
              if (more) {
                mma_kk<D>(one, t_s, desc_k(qs + t * C::TILE_BYTES), desc_k(stage(kn)), id_s);
                commit1(one, &s_full[t]);
                if (t == f.nt - 1) {
                  commit1(one, &kv_empty[kn % ST]);
                  if (i + 2 == f.n) commit1(one, q_empty);
                }
              }
            }
            if (!ok) break;
            si += 2;
          }
          if (!ok) break;
          for (int t = 0; t < f.nt; ++t) cnt[t] += uint32_t(f.n);
        }
        unit_done(sched, k);
      }
      // no commit may arrive after the block has left
      commit1(one, all_done);
      wait_for(all_done, 0, abort_flag, 0x2207);
    } else if (warp == 10) {
      // -------------------------------------------------------------- units and their lists
      run_scheduler(sched, abort_flag, 0x2401, [&](int x, int y, int z, uint32_t slot) {
        const FwdUnit f = fwd_unit(prm, Unit{x, y, z, 0});
        if (int(lane) < f.nt * (D / 64)) {
          const int t = int(lane) / (D / 64);
          prefetch_l2_4d(&tm_q, int(lane) % (D / 64) * 64, t ? f.head[1] : f.head[0], t ? f.pos[1] : f.pos[0], f.b);
        }
        if (!p.has_docs) return 0;
        const DocRange qd = warp_doc_range(p.qdoc + (size_t)f.b * p.sq + f.pos[0], f.last_pos - f.pos[0] + 1, lane);
        const int hi = max(0, row_limit(p, f.last_pos, f.pre) + TILE - 1) / TILE;
        const int t1 = min(min(p.n_tiles, f.t0 + p.tiles_per_split), hi);
        int n = 0;
        for (int t = f.t0; t < t1; t += 32) {
          int st = kStSkip;
          bool scrub = false;
          if (t + int(lane) < t1) {
            const int j0 = (t + int(lane)) * TILE;
            const DocRange kd = p.krange[(size_t)f.b * p.n_tiles + t + lane];
            // keys behind the end are masked like unseen ones
            st = pair_state(p, f.pre, f.pos[0], f.last_pos, j0, j0 + TILE - 1, qd, kd);
            scrub = kd.neg != 0;
          }
          n = list_append(lists + slot * kMaxList, n, t - f.t0 + int(lane), st, scrub, lane);
        }
        return n;
      });
    }
  } else {
    // ---------------------------------------------------------------- softmax, one thread a row
    regs_grow();
    const int t = warp >> 2;
    const uint32_t t_lane = uint32_t((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + t_lane + t * TILE, t_o = tmem + t_lane + 2 * TILE + t * D;
    const int row = int(warp & 3) * 32 + int(lane);
    const uint32_t stage = smem_u32(smem + C::OFF_STAGE) + warp * 2048;
    // scores that are only scaled stay raw and are scaled inside the exponent
    const float c = BIAS || CAP ? 1.f : p.scale_log2;
    const float grow = fminf(8.f / c, 3e38f);
    const TanhSmall tanh_small(p);
    uint32_t cnt = 0;   // tiles so far
    for (uint32_t k = 0; next_unit(sched, k, u, abort_flag, 0x2304); ++k) {
      const FwdUnit f = fwd_unit(prm, u);
      if (!DUO && t >= f.nt) {
        unit_done(sched, k);
        continue;
      }
      const uint16_t* list = lists + (k & 1) * kMaxList;
      int pos, head;
      bool valid;
      if (prm.packed) {
        const int r = p.divG.div(row);
        pos = (t && !DUO ? f.pos[1] : f.pos[0]) + r;
        head = f.head[0] + row - r * p.G;
        valid = r < prm.pos_per_tile && pos < p.sq;
      } else {
        pos = (t && !DUO ? f.pos[1] : f.pos[0]) + row;
        head = t && !DUO ? f.head[1] : f.head[0];
        valid = pos < p.sq;
      }
      const int lim = valid ? row_limit(p, pos, f.pre) : 0;
      const int qd = (valid && p.has_docs) ? __ldg(p.qdoc + (size_t)f.b * p.sq + pos) : -1;
      const bool any_valid = __any_sync(0xffffffffu, valid);   // warps of padding rows only pass barriers
      const float slope2 = (BIAS && valid) ? __ldg(p.slopes + head) * kLog2e : 0.f;

      float mref = -INFINITY;   // reference maximum, in units of 1 / c
      float l = 0.f;
      bool ok = true;
      const int n = DUO ? (f.n + 1 - t) >> 1 : f.n;   // tiles of these warps
      for (int i = 0; i < n; ++i) {
        const int ti = DUO ? 2 * i + t : i;
        const uint32_t ent = p.has_docs ? list[ti] : 0u;
        const int j0 = (f.t0 + (p.has_docs ? int(ent & kEntTile) : ti)) * TILE;
        const bool masked = p.has_docs ? (ent & kEntMask) != 0 : j0 + TILE > f.lim0;
        // which keys this row sees.  Before the wait, since the documents' numbers come from far away
        // (8192 packed positions 425 -> 390 us)
        uint32_t see[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
        if (__builtin_expect(masked, 0)) {
          if (p.has_docs) {
            int ids[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const int j = j0 + g * 32 + int(lane);
              ids[g] = j < p.skv ? __ldg(p.kdoc + (size_t)f.b * p.skv + j) : -1;
            }
            same_ids<4>(ids, qd, see);
          }
#pragma unroll
          for (int g = 0; g < 4; ++g) see[g] &= low_bits(lim - j0 - g * 32);
        }
        ok = wait_for(&s_full[t], (cnt + i) & 1, abort_flag, 0x2301);
        if (!ok) break;
        tc_fence_after();
        // every completion of o_done is waited for once, so its parity cannot be mistaken
        bool o_seen = i == 0;
        if (__builtin_expect(any_valid, 1)) {
          // Three ways through a row, by what has to be done to its scores:
          //   nothing but a mask, or a bias that is linear along it: 128 scores stay in registers;
          //   cap alone: the maximum is the tanh of the raw scores' maximum, and the tanh is
          //     taken next to the exponentials, which use other units;
          //   anything else: scores are rewritten in TMEM, 32 at a time, then read again.
          // (All of it on 128 scores in registers spilled, and a row read twice cost the plain
          // case 10 % of the 4096x4096 prompt.)
          auto hide = [](uint32_t (&x)[32], uint32_t seen) {   // -inf to the keys that are not seen
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((seen >> e) & 1u)) x[e] = 0xff800000u;
          };
          // 32 scores from column 32 g on: cap, bias, mask (log2 units / c, -inf where not seen)
          auto modify = [&](uint32_t (&x)[32], int g) {
            if (CAP) {
              if (cap_small(p, highest_abs(x), p.has_docs && qd < 0)) cap32<true>(p, tanh_small, x);
              else cap32<false>(p, tanh_small, x);
            }
            if (BIAS) {
              const float d0 = float(pos + p.off - j0 - g * 32), sl = CAP ? 1.f : p.scale_log2;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                x[e] = __float_as_uint(fmaf(__uint_as_float(x[e]), sl, -slope2 * fabsf(d0 - float(e))));
            }
            if (__builtin_expect(masked, 0)) hide(x, g == 0 ? see[0] : g == 1 ? see[1] : g == 2 ? see[2] : see[3]);
          };
          auto highest = [](const uint32_t (&x)[32]) {
            float y[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              y[h] = fmaxf(__uint_as_float(x[16 * h]), __uint_as_float(x[16 * h + 1]));
#pragma unroll
              for (int e = 2; e < 16; e += 2)
                y[h] = fmaxf(y[h], fmaxf(__uint_as_float(x[16 * h + e]), __uint_as_float(x[16 * h + e + 1])));
            }
            return fmaxf(y[0], y[1]);
          };
          const bool linear = BIAS && __all_sync(0xffffffffu, pos + p.off >= j0 + TILE - 1);
          const bool in_regs = !CAP && (!BIAS || linear);
          const bool late_cap = CAP && !BIAS && !masked;
          uint32_t x[4][32];
          float m;
          bool small = false;
          if (in_regs || late_cap) {
#pragma unroll
            for (int g = 0; g < 4; ++g) tmem_ld32(t_s + g * 32, x[g]);
            tmem_wait_ld();
            if (BIAS) {
              // the distance itself runs along the row (exact below 2^24 positions): with slope2 * position
              // taken out of the product a bias was off by the rounding of up to 254 slopes, however near its key
              const uint64_t c2 = f2(p.scale_log2, p.scale_log2), s2 = f2(slope2, slope2), two = f2(2.f, 2.f);
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const int d = j0 + g * 32 - pos - p.off;
                uint64_t t = f2(float(d), float(d + 1));
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                  float u, v;
                  f2_split(f2_fma(t, s2, f2_mul(f2(__uint_as_float(x[g][e]), __uint_as_float(x[g][e + 1])), c2)), u, v);
                  x[g][e] = __float_as_uint(u);
                  x[g][e + 1] = __float_as_uint(v);
                  t = f2_add(t, two);
                }
              }
            }
            if (!CAP && __builtin_expect(masked, 0)) {
#pragma unroll
              for (int g = 0; g < 4; ++g) hide(x[g], see[g]);
            }
            m = fmaxf(fmaxf(highest(x[0]), highest(x[1])), fmaxf(highest(x[2]), highest(x[3])));
            if (CAP)
              small = cap_small(p, fmaxf(fmaxf(highest_abs(x[0]), highest_abs(x[1])),
                                         fmaxf(highest_abs(x[2]), highest_abs(x[3]))), false);   // not masked: no padding
            if (CAP) m = cap1(p, tanh_small, m);   // the tanh grows with its argument
          } else if constexpr (CAP || BIAS) {
            m = -INFINITY;
#pragma unroll 1
            for (int g = 0; g < 4; ++g) {
              uint32_t y[32];
              __syncwarp();
              tmem_ld32(t_s + g * 32, y);
              tmem_wait_ld();
              modify(y, g);
              m = fmaxf(m, highest(y));
              tmem_st16(t_s + g * 32, *reinterpret_cast<uint32_t (*)[16]>(&y[0]));
              tmem_st16(t_s + g * 32 + 16, *reinterpret_cast<uint32_t (*)[16]>(&y[16]));
            }
            tmem_wait_st();
          }
          if (__builtin_expect(__any_sync(0xffffffffu, m > mref + grow), 0)) {
            const float mnew = fmaxf(mref, m);
            const float fac = mref == mnew ? 1.f : ex2((mref - mnew) * c);   // 0 from a reference of -inf
            mref = mnew;
            l *= fac;
            if (i > 0) {
              ok = wait_for(&o_done[t], (cnt + i - 1) & 1, abort_flag, 0x2302);
              if (!ok) break;
              o_seen = true;
              tc_fence_after();
#pragma unroll 1
              for (int x = 0; x < D / 16; ++x) {
                uint32_t o[16];
                tmem_ld16(t_o + x * 16, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fac);
                tmem_st16(t_o + x * 16, o);
              }
              tmem_wait_st();
            }
          }
          const float nm = mref == -INFINITY ? 0.f : -mref * c;
          const uint64_t c2 = f2(c, c), nm2 = f2(nm, nm);
          uint64_t sum0 = 0, sum1 = 0;
          // weights of 32 keys, to 16 columns.  TR 0: of scores; 1, 2: of raw scores to be capped
          auto weigh = [&](const uint32_t (&y)[32], uint32_t column, auto tr_tag) {
            constexpr int TR = decltype(tr_tag)::value;
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              float a[4];
#pragma unroll
              for (int z = 0; z < 4; ++z) a[z] = __uint_as_float(y[e + z]);
              if (TR) {
                cap4<TR == 1>(p, tanh_small, a, nm);
              } else {
                f2_split(f2_fma(f2(a[0], a[1]), c2, nm2), a[0], a[1]);
                f2_split(f2_fma(f2(a[2], a[3]), c2, nm2), a[2], a[3]);
              }
#pragma unroll
              for (int z = 0; z < 4; ++z) a[z] = ex2(a[z]);
              sum0 = f2_add(sum0, f2(a[0], a[1]));
              sum1 = f2_add(sum1, f2(a[2], a[3]));
              w[e / 2] = pack2<F16>(a[0], a[1]);
              w[e / 2 + 1] = pack2<F16>(a[2], a[3]);
            }
            tmem_st16(t_s + column, w);
          };
          // the weights of 64 keys are written: the second product may take them
          auto hand_over = [&](int h) {
            tmem_wait_st();
            tc_fence_before();
            if (!o_seen) {
              ok = wait_for(&o_done[t], (cnt + i - 1) & 1, abort_flag, 0x2305);
              o_seen = true;
            }
            __syncwarp();
            if (lane == 0 && ok) mbar_arrive(&p_ready[2 * t + h]);
          };
          if (in_regs) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              weigh(x[g], g * 16, std::integral_constant<int, 0>{});
              if (g & 1) hand_over(g >> 1);
            }
          } else if constexpr (CAP || BIAS) {
            auto again = [&](auto tr_tag) {
#pragma unroll 1
              for (int h = 0; h < 2; ++h) {
#pragma unroll 1
                for (int g = 2 * h; g < 2 * h + 2; ++g) {
                  uint32_t y[32];
                  __syncwarp();
                  tmem_ld32(t_s + g * 32, y);
                  tmem_wait_ld();
                  weigh(y, g * 16, tr_tag);
                }
                hand_over(h);
              }
            };
            if (CAP && late_cap && small) again(std::integral_constant<int, 1>{});
            else if (CAP && late_cap) again(std::integral_constant<int, 2>{});
            else again(std::integral_constant<int, 0>{});
          }
          if (!ok) break;
          float x0, x1, y0, y1;
          f2_split(sum0, x0, x1);
          f2_split(sum1, y0, y1);
          l += (x0 + x1) + (y0 + y1);
        } else {
          if (!o_seen) ok = wait_for(&o_done[t], (cnt + i - 1) & 1, abort_flag, 0x2306);
          if (!ok) break;
          tc_fence_before();
          if (lane == 0) {
            mbar_arrive(&p_ready[2 * t]);
            mbar_arrive(&p_ready[2 * t + 1]);
          }
        }
      }
      // ---- epilogue: o / l, and the row statistic
      if (ok && n > 0) ok = wait_for(&o_done[t], (cnt + n - 1) & 1, abort_flag, 0x2303);
      if (!ok) break;
      cnt += uint32_t(n);
      if (any_valid) {
        tc_fence_after();
        const bool empty = l == 0.f;
        const float inv = empty ? 0.f : 1.f / l;
        const float lse = empty ? -INFINITY : (mref * c + log2f(l)) * kLn2;
        const size_t rowi = ((size_t)f.b * p.H + head) * p.sq + pos;
        const size_t ri = (size_t)(DUO ? 2 * f.split + t : f.split) * p.bs * p.H * p.sq + rowi;
        if (valid) (p.splits > 1 ? prm.part_lse + ri : prm.lse + rowi)[0] = lse;
        uint8_t* dst = static_cast<uint8_t*>(prm.o) + (((size_t)f.b * p.sq + pos) * p.H + head) * (D * 2);
        // (64 columns a load would hide more of TMEM's latency, but leaves the loop above fewer
        // registers: 7 % of the 4096x4096 prompt)
#pragma unroll 1
        for (int x = 0; x < D / 32; ++x) {
          uint32_t o[32];
          __syncwarp();
          if (n > 0) {
            tmem_ld32(t_o + x * 32, o);
            tmem_wait_ld();
          }
          if (DUO || p.splits > 1) {   // DUO leaves two parts at least
            if (valid) {
              float4* part = reinterpret_cast<float4*>(prm.part_o + ri * D + x * 32);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                part[e] = empty ? make_float4(0.f, 0.f, 0.f, 0.f)
                                : make_float4(__uint_as_float(o[4 * e]) * inv, __uint_as_float(o[4 * e + 1]) * inv,
                                              __uint_as_float(o[4 * e + 2]) * inv, __uint_as_float(o[4 * e + 3]) * inv);
            }
          } else {
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
              w[e] = empty ? 0u : pack2<F16>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
            if (prm.packed) {   // (position, head) rows are no box
              if (valid) write_row(w, dst + x * 64, prm.wide != 0);
            } else {
              store_rows(stage, &tm_o, w, x * 32, head, pos - int(lane), f.b, lane);
            }
          }
        }
        tc_fence_before();   // the next unit's first product overwrites the accumulator
      }
      unit_done(sched, k);
    }
    if (lane == 0) bulk_wait_all0();   // no store may outlive the block
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  report_error(abort_flag, p.err);
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the splits of every row: o = sum_s 2^(lse_s - lse) o_s.  One warp a row; the sum
// over splits runs in order, so equal inputs give equal bits.  Bound by its launch and the latency of
// its loads: 6 us for 320 rows of 8 parts, 8 us for 3080 rows of 9.
template <int D, bool F16>
__global__ void __launch_bounds__(256) fwd_join_kernel(const FwdParams prm) {
  wait_for_previous();
  const Params& p = prm.c;
  const long long rows = (long long)p.bs * p.H * p.sq;
  const long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (r >= rows) return;
  float mx = -INFINITY;
  bool nan = false;
  for (int s = lane; s < p.splits; s += 32) {
    const float x = prm.part_lse[(long long)s * rows + r];
    nan = nan || x != x;
    mx = fmaxf(mx, x);
  }
#pragma unroll
  for (int k = 16; k; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
  if (__any_sync(0xffffffffu, nan)) mx = 0.f;   // the row is NaN: its weights below are too
  constexpr int N = D / 32;   // elements of a lane
  float acc[N] = {}, l = 0.f;
  if (mx != -INFINITY) {
    for (int s = 0; s < p.splits; ++s) {
      const float w = ex2((prm.part_lse[(long long)s * rows + r] - mx) * kLog2e);
      const float* src = prm.part_o + ((long long)s * rows + r) * D + lane * N;
      l += w;
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = fmaf(w, src[e], acc[e]);
    }
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);   // NaN stays NaN
  const long long bh = r / p.sq, pos = r - bh * p.sq, b = bh / p.H, h = bh - b * p.H;
  uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(prm.o) + ((b * p.sq + pos) * p.H + h) * (D * 2)) +
                  lane * (N / 2);
#pragma unroll
  for (int e = 0; e < N / 2; ++e) dst[e] = pack2<F16>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  if (lane == 0) prm.lse[r] = mx == -INFINITY ? -INFINITY : mx + logf(l);
}

// The tensor maps of a call.
struct FwdMaps {
  CUtensorMap q, k, v, o;
};
// fused_fwd.cu, fused_token.cu (units of one tile)
int launch_fwd(const FwdParams& f, const FwdMaps& m, int d, bool f16, bool cap, cudaStream_t s);
int launch_token(const FwdParams& f, const FwdMaps& m, int d, bool f16, bool cap, cudaStream_t s);

template <bool DUO, int D, bool F16, bool CAP, bool BIAS>
static int launch_one(const FwdParams& f, const FwdMaps& m, cudaStream_t stream) {
  using C = FwdCfg<D, DUO>;
  const auto kern = fwd_kernel<D, F16, CAP, BIAS, DUO>;
  const int rc = prepare_kernel(reinterpret_cast<const void*>(kern), C::SMEM_BYTES);
  if (rc) return rc;
  const dim3 grid(unsigned(f.blocks_q) * f.head_slots, f.c.bs, f.cta_splits);
  return launch_kernel(kern, grid, kThreads, C::SMEM_BYTES, stream, f.c.has_docs && f.c.n_tiles > 0, m.q, m.k, m.v, m.o, f);
}
template <bool DUO, int D, bool F16>
static int launch_scores(const FwdParams& f, const FwdMaps& m, bool cap, cudaStream_t s) {
  if (f.c.slopes)
    return cap ? launch_one<DUO, D, F16, true, true>(f, m, s) : launch_one<DUO, D, F16, false, true>(f, m, s);
  return cap ? launch_one<DUO, D, F16, true, false>(f, m, s) : launch_one<DUO, D, F16, false, false>(f, m, s);
}
template <bool DUO>
static int launch_any(const FwdParams& f, const FwdMaps& m, int d, bool f16, bool cap, cudaStream_t s) {
  if (d == 128) return f16 ? launch_scores<DUO, 128, true>(f, m, cap, s) : launch_scores<DUO, 128, false>(f, m, cap, s);
  return f16 ? launch_scores<DUO, 64, true>(f, m, cap, s) : launch_scores<DUO, 64, false>(f, m, cap, s);
}

}  // namespace fused
}  // namespace attn_bwd
