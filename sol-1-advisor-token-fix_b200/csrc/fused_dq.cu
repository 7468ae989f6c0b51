// fused_dq.cu — gradient of the queries (see fused_bwd.cuh).  8192 packed positions in documents of
// about 2500, 80 + 8 heads of 128: 653 us; 48 sequences of 640, capped: 1340 us (units of three key
// tiles, where beginning and ending a unit takes about 4 of its 10 us).
#include "fused_bwd.cuh"
#include "fused_host.h"

namespace attn_bwd {
namespace fused {

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
template <int D, bool F16, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kThreads, 1)
dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
          const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
          const __grid_constant__ CUtensorMap tm_dq,   // (d, s, h, b), box (32, 32, 1, 1)
          const BwdParams prm) {
  using C = BwdCfg<D>;
  constexpr int ST = C::ST;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const BwdShared sh = bwd_shared<D>(smem_raw);
  const Params& p = prm.c;
  const uint32_t warp = warp_id(), lane = lane_id();
  const uint32_t tmem = bwd_begin(sh, ST, 9, &tm_q, &tm_do, &tm_k, &tm_v);
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
            const uint32_t t_s = tmem + (it & 1) * TILE;
            if (!(ok = wait_for(&sh.ds_ready[0], it & 1, sh.abort_flag, 0x4206))) break;
            tc_fence_after();
            mma_tn_part<D, 0>(one, t_dq, t_s, t_s + 64, desc_mn(stage(2 * it)), id_g, i > 0);
            if (!(ok = wait_for(&sh.ds_ready[1], it & 1, sh.abort_flag, 0x420a))) break;
            tc_fence_after();
            // first, since the next load of keys waits for their tile
            mma_tn_part<D, 1>(one, t_dq, t_s, t_s + 64, desc_mn(stage(2 * it)), id_g, true);
            commit1(one, &sh.empty[(2 * it) % ST]);
            if (i + 1 == f.n) commit1(one, sh.done);
            if (i + 1 < f.n) {
              mma_kk<D>(one, t_dp, dos, desc_k(stage(2 * it + 3)), id_s);
              commit1(one, sh.dp_full);
              commit1(one, &sh.empty[(2 * it + 3) % ST]);
              if (i + 2 == f.n) commit1(one, sh.res_empty);   // the last scores were issued before
            }
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
        const DqUnit f = dq_unit(prm, Unit{x, y, z, 0});
        if (int(lane) < 2 * (D / 64))
          prefetch_l2_4d(int(lane) & 1 ? &tm_do : &tm_q, (int(lane) >> 1) * 64, f.r0, f.h, f.b);
        auto prefetch_o = [&](int tiles) {   // rows of one key tile read no o
          if (tiles > 1)
            for (int r = f.r0 + int(lane); r <= f.r1; r += 32)
              for (int c = 0; c < D * 2; c += 128)
                prefetch_l2(prm.o + (((size_t)f.b * p.sq + r) * p.H + f.h) * (D * 2) + c);
        };
        if (!p.has_docs) {
          prefetch_o(f.n);
          return 0;
        }
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
        prefetch_o(n);
        return n;
      });
    }
  } else {
    // ---------------------------------------------------------------- weights: one query a thread, 64 keys
    regs_grow();
    const uint32_t stage = smem_u32(sh.smem + C::OFF_STAGE) + warp * 2048;
    constexpr int LR = D / 16;   // 16-byte words of half a row
    const TanhSmall tanh_small(p);
    const int half = int(warp) >> 2;
    const uint32_t t_lane = uint32_t((warp & 3) * 32) << 16;
    const uint32_t dp = t_dp + t_lane + half * 64;
    uint32_t it = 0, di = 0, met = 0;
    bool ok = true;
    for (uint32_t k = 0; ok && next_unit(sh.sched, k, u, sh.abort_flag, 0x4304); ++k) {
      const DqUnit f = dq_unit(prm, u);
      const uint16_t* list = sh.lists + (k & 1) * kMaxList;
      const int row = f.r0 + int(warp & 3) * 32 + int(lane);
      const bool valid = row < p.sq, any_valid = row - int(lane) < p.sq;
      const size_t ri = ((size_t)f.b * p.H + f.h) * prm.sq_pad + row;   // padded to whole tiles
      const float lse = valid ? __ldg(prm.lse + ((size_t)f.b * p.H + f.h) * p.sq + row) : -INFINITY;
      // o of these rows, this half of the columns, for delta: the lanes of a group of LR read one row's
      // part together (a lane reading its own row's would touch 32 lines a load).  Used, like
      // lse, only after the wait for the first scores.
      uint4 ov[LR];
      if (f.n > 1) {
#pragma unroll
        for (int c = 0; c < LR; ++c) {
          const int r = min(f.r1, f.r0 + int(warp & 3) * 32 + c * (32 / LR) + int(lane) / LR);
          ov[c] = __ldg(reinterpret_cast<const uint4*>(prm.o + (((size_t)f.b * p.sq + r) * p.H + f.h) * (D * 2) + half * D) +
                        int(lane) % LR);
        }
      }
      bool none = false;       // the row sees nothing
      float nlse = 0.f;
      uint64_t nd2 = 0;
      const int lim = valid ? row_limit(p, row, f.pre) : 0;
      const int qd = (valid && p.has_docs) ? __ldg(p.qdoc + (size_t)f.b * p.sq + row) : -1;
      const float slope2 = BIAS ? __ldg(p.slopes + f.h) * kLog2e : 0.f;
      if (f.n == 0 && half == 0) {   // no tile, so no key tile asks for these
        prm.nlse[ri] = -INFINITY;
        prm.ndelta[ri] = 0.f;
      }
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
        if (i == 0) {
          none = lse == -INFINITY;
          nlse = none ? -INFINITY : -lse * kLog2e;
        }
        uint32_t w[2][32];
#pragma unroll
        for (int y = 0; y < 2; ++y) tmem_ld32(st + y * 32, w[y]);
        tmem_wait_ld();
        const float dist0 = float(row + p.off - j0);
        auto phase = [&](auto small_tag) {
          constexpr bool SMALL = decltype(small_tag)::value;
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
              weights4<CAP, SMALL>(p, tanh_small, x, add, m);
#pragma unroll
              for (int z = 0; z < 4; ++z) w[y][e + z] = __float_as_uint(m[z]);
            }
        };
        const bool small = CAP && cap_small(p, fmaxf(highest_abs(w[0]), highest_abs(w[1])), p.has_docs && qd < 0);
        if (!CAP || f.n > 1) {   // (below otherwise)
          if (CAP && small) phase(std::true_type{});
          else phase(std::false_type{});
        }
        if (i == 0 && f.n > 1) {
          // delta of the row: each half of the warps takes half of the columns
          ok = wait_for(sh.res_full, di & 1, sh.abort_flag, 0x4305);
          if (!ok) break;
          const int r = int(warp & 3) * 32 + int(lane);
          float* part = reinterpret_cast<float*>(sh.smem + C::OFF_STAT) + (k & 1) * (4 * TILE);
#pragma unroll
          for (int c = 0; c < LR; ++c) {
            const int rr = int(warp & 3) * 32 + c * (32 / LR) + int(lane) / LR, cg = half * LR + int(lane) % LR;
            const uint4 g = lds128(smem_u32(sh.smem + C::OFF_A + C::TILE_BYTES) + (cg >> 3) * (TILE * 128) + rr * 128 +
                                   (((cg & 7) ^ (rr & 7)) << 4));
            const uint32_t gs[4] = {g.x, g.y, g.z, g.w}, os[4] = {ov[c].x, ov[c].y, ov[c].z, ov[c].w};
            float d = 0.f;
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const float2 u = unpack2<F16>(gs[z]), v = unpack2<F16>(os[z]);
              d = fmaf(u.x, v.x, d);
              d = fmaf(u.y, v.y, d);
            }
#pragma unroll
            for (int m = LR / 2; m; m >>= 1) d += __shfl_xor_sync(0xffffffffu, d, m);
            if (int(lane) % LR == 0) part[half * TILE + rr] = d;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(sh.res_empty);
          ok = meet(&sh.pair[warp & 3], met, sh.abort_flag, 0x4306);   // the two warps of these rows
          if (!ok) break;
          const float d = part[r] + part[TILE + r];
          const float nd = none ? 0.f : -d;
          nd2 = f2(nd, nd);
          if (half == 0) {
            prm.nlse[ri] = nlse;
            prm.ndelta[ri] = nd;
          }
        }
        // masked scores are taken out of ds below
        ok = wait_for(sh.dp_full, it & 1, sh.abort_flag, 0x4302);
        if (!ok) break;
        tc_fence_after();
        if (f.n == 1) {
          // All of the row's weights are here: delta = sum(p dp) / sum(p), without o, whose 16 bits cost
          // delta most where a row sees few keys and ds is small beside it.  (Rows of more tiles would
          // need their tiles twice: a fifth of the pass.)
          uint64_t pd2 = f2(0.f, 0.f), ps2 = f2(0.f, 0.f);
          auto whole = [&](auto small_tag) {
            constexpr bool SMALL = decltype(small_tag)::value;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              uint32_t d[32];
              tmem_ld32(dp + y * 32, d);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                float x[4];
#pragma unroll
                for (int z = 0; z < 4; ++z) x[z] = __uint_as_float(w[y][e + z]);
                if (CAP) {
                  float add[4], m[4];
#pragma unroll
                  for (int z = 0; z < 4; ++z)
                    add[z] = BIAS ? fmaf(-slope2, fabsf(dist0 - float(y * 32 + e + z)), nlse) : nlse;
                  weights4<CAP, SMALL>(p, tanh_small, x, add, m);
#pragma unroll
                  for (int z = 0; z < 4; ++z) w[y][e + z] = __float_as_uint(m[z]);
                }
#pragma unroll
                for (int z = 0; z < 4; ++z)
                  if (!((see[y] >> (e + z)) & 1u)) {
                    x[z] = 0.f;
                    d[e + z] = 0u;
                  }
#pragma unroll
                for (int z = 0; z < 4; z += 2) {
                  pd2 = f2_fma(f2(x[z], x[z + 1]), f2(d[e + z], d[e + z + 1]), pd2);
                  ps2 = f2_add(ps2, f2(x[z], x[z + 1]));
                }
              }
            }
          };
          if (CAP && small) whole(std::true_type{});
          else whole(std::false_type{});
          float a0, a1, b0, b1;
          f2_split(pd2, a0, a1);
          f2_split(ps2, b0, b1);
          const int r = int(warp & 3) * 32 + int(lane);
          float2* part = reinterpret_cast<float2*>(sh.smem + C::OFF_STAT) + (k & 1) * (2 * TILE);
          part[half * TILE + r] = make_float2(a0 + a1, b0 + b1);
          if (lane == 0) mbar_arrive(sh.res_empty);
          ok = meet(&sh.pair[warp & 3], met, sh.abort_flag, 0x4307);
          if (!ok) break;
          const float2 u = part[r], v = part[TILE + r];
          const float nd = none ? 0.f : -(u.x + v.x) / (u.y + v.y);
          nd2 = f2(nd, nd);
          if (half == 0) {
            prm.nlse[ri] = nlse;
            prm.ndelta[ri] = nd;
          }
        }
        auto gradients = [&](auto mask_tag) {
          constexpr bool MASK = decltype(mask_tag)::value;
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t d[32], pk[16];
            tmem_ld32(dp + y * 32, d);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float a0, a1;
              f2_split(f2_mul(f2(w[y][e], w[y][e + 1]), f2_add(f2(d[e], d[e + 1]), nd2)), a0, a1);
              if (MASK) {
                if (!((see[y] >> e) & 1u)) a0 = 0.f;
                if (!((see[y] >> (e + 1)) & 1u)) a1 = 0.f;
              }
              pk[e / 2] = pack2<F16>(a0, a1);
            }
            tmem_st16(st + y * 16, pk);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.ds_ready[y]);
          }
        };
        if (__builtin_expect(masked, 0)) gradients(std::true_type{});
        else gradients(std::false_type{});
      }
      if (!ok) break;
      // ---- epilogue: each half of the warps writes half of the columns
      if (f.n > 0) {
        ok = wait_for(sh.done, di & 1, sh.abort_flag, 0x4303);
        if (!ok) break;
        ++di;
      }
      tc_fence_after();
      uint32_t v[D / 64][32];
#pragma unroll
      for (int x = 0; x < D / 64; ++x)
#pragma unroll
        for (int e = 0; e < 32; ++e) v[x][e] = 0u;
      __syncwarp();
      if (f.n > 0) {   // all loads first: TMEM answers slowly while the tensor cores write to it
#pragma unroll
        for (int x = 0; x < D / 64; ++x) tmem_ld32(t_dq + t_lane + half * (D / 2) + x * 32, v[x]);
        tmem_wait_ld();
      }
#pragma unroll
      for (int x = 0; x < D / 64; ++x) {
        uint32_t o[16];
#pragma unroll
        for (int e = 0; e < 16; ++e)
          o[e] = pack2<F16>(__uint_as_float(v[x][2 * e]) * p.scale, __uint_as_float(v[x][2 * e + 1]) * p.scale);
        if (any_valid) store_rows(stage, &tm_dq, o, half * (D / 2) + x * 32, row - int(lane), f.h, f.b, lane);
      }
      tc_fence_before();   // the next unit's first product overwrites the accumulator
      unit_done(sh.sched, k);
    }
    if (lane == 0) bulk_wait_all0();   // no store may outlive the block
    __syncwarp();
  }
  bwd_end(sh, tmem, p.err);
}

template <int D, bool F16, bool CAP, bool BIAS>
static int launch(const BwdParams& f, const CUtensorMap& q, const CUtensorMap& go, const CUtensorMap& k,
                  const CUtensorMap& v, const CUtensorMap& dq, cudaStream_t s) {
  using C = BwdCfg<D>;
  const auto kern = dq_kernel<D, F16, CAP, BIAS>;
  const int rc = prepare_kernel(reinterpret_cast<const void*>(kern), C::SMEM_BYTES);
  if (rc) return rc;
  const dim3 grid(unsigned(f.c.n_tiles) * f.c.H, f.c.bs);
  return launch_kernel(kern, grid, kThreads, C::SMEM_BYTES, s, f.c.has_docs, q, go, k, v, dq, f);
}

int launch_dq(const BwdParams& f, const CUtensorMap& q, const CUtensorMap& go, const CUtensorMap& k,
              const CUtensorMap& v, const CUtensorMap& dq, int d, bool f16, bool cap, cudaStream_t s) {
  const bool bias = f.c.slopes != nullptr;
#define ATTN_BWD_PICK(DD, FF)                                                                                   \
  if (d == DD && f16 == FF)                                                                                     \
    return cap ? (bias ? launch<DD, FF, true, true>(f, q, go, k, v, dq, s) : launch<DD, FF, true, false>(f, q, go, k, v, dq, s)) \
               : (bias ? launch<DD, FF, false, true>(f, q, go, k, v, dq, s) : launch<DD, FF, false, false>(f, q, go, k, v, dq, s));
  ATTN_BWD_PICK(128, false)
  ATTN_BWD_PICK(128, true)
  ATTN_BWD_PICK(64, false)
  ATTN_BWD_PICK(64, true)
#undef ATTN_BWD_PICK
  return ATTN_BWD_EUNSUPPORTED;
}

}  // namespace fused
}  // namespace attn_bwd
