// fused_dkv.cu — gradients of keys and values (see fused_bwd.cuh).  8192 packed positions in documents of
// about 2500, 80 + 8 heads of 128: 878 us; 48 sequences of 640, capped: 1085 us.
#include "fused_bwd.cuh"
#include "fused_host.h"

namespace attn_bwd {
namespace fused {

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

template <int D, bool F16, bool CAP, bool BIAS>
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
  const uint32_t tmem = bwd_begin(sh, ST, 1, &tm_q, &tm_do, &tm_k, &tm_v);
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
            if (!(ok = wait_for(&sh.p_ready[0], it & 1, sh.abort_flag, 0x3205))) break;
            tc_fence_after();
            mma_tn_part<D, 0>(one, t_dv, t_st, t_st + 64, desc_mn(stage(2 * it + 1)), id_g, i > 0);
            if (!(ok = wait_for(&sh.p_ready[1], it & 1, sh.abort_flag, 0x3200))) break;
            tc_fence_after();
            mma_tn_part<D, 1>(one, t_dv, t_st, t_st + 64, desc_mn(stage(2 * it + 1)), id_g, true);
            commit1(one, &sh.empty[(2 * it + 1) % ST]);
            if (more) {
              mma_kk<D>(one, t_st, ks, desc_k(stage(2 * it + 2)), id_s);
              commit1(one, &sh.s_full[0]);
            }
            if (more && !(ok = arrived(2 * it + 3, t, 0x3206))) break;
            if (!(ok = wait_for(&sh.ds_ready[0], it & 1, sh.abort_flag, 0x3207))) break;
            tc_fence_after();
            mma_tn_part<D, 0>(one, t_dk, t_dp, t_dp + 64, desc_mn(stage(2 * it)), id_g, i > 0);
            if (!(ok = wait_for(&sh.ds_ready[1], it & 1, sh.abort_flag, 0x320a))) break;
            tc_fence_after();
            mma_tn_part<D, 1>(one, t_dk, t_dp, t_dp + 64, desc_mn(stage(2 * it)), id_g, true);
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
        const DkvUnit f = dkv_unit(prm, Unit{x, y, z, 0});
        if (int(lane) < 2 * (D / 64))
          prefetch_l2_4d(int(lane) & 1 ? &tm_v : &tm_k, (int(lane) >> 1) * 64, f.j0, f.kvh, f.b);
        if (!p.has_docs) return 0;
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
    const TanhSmall tanh_small(p);
    const int half = int(warp) >> 2;
    const uint32_t t_lane = uint32_t((warp & 3) * 32) << 16;
    const uint32_t st = t_st + t_lane + half * 64, dp = t_dp + t_lane + half * 64;
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
        const uint32_t stat = smem_u32(sh.smem + C::OFF_STAT + (it & 1) * (2 * TILE * 4) + half * 256);
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
        const float slope2 = BIAS ? __ldg(p.slopes + f.kvh * p.G + g) * kLog2e : 0.f;
        const float dist0 = float(r0 + p.off - j);
        // the rows' statistics are read before the wait for the scores: shared memory answers slowly
        // while the tensor cores read from it
        ok = wait_for(&sh.full[(2 * it) % ST], ((2 * it) / ST) & 1, sh.abort_flag, 0x3302);
        if (!ok) break;
        float4 nl4[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) nl4[e] = lds_f4(stat + e * 16);
        ok = wait_for(&sh.s_full[0], it & 1, sh.abort_flag, 0x3301);
        if (!ok) break;
        tc_fence_after();
        uint32_t w[2][32];   // scores, then what ds is multiplied by
#pragma unroll
        for (int y = 0; y < 2; ++y) tmem_ld32(st + y * 32, w[y]);
        tmem_wait_ld();
        auto phase = [&](auto mask_tag, auto small_tag) {
          constexpr bool MASK = decltype(mask_tag)::value, SMALL = decltype(small_tag)::value;
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 nl = nl4[y * 8 + e / 4];
              float add[4] = {nl.x, nl.y, nl.z, nl.w}, x[4], m[4];
#pragma unroll
              for (int z = 0; z < 4; ++z) {
                x[z] = __uint_as_float(w[y][e + z]);
                if (BIAS) add[z] = fmaf(-slope2, fabsf(dist0 + float(y * 32 + e + z)), add[z]);
              }
              weights4<CAP, SMALL>(p, tanh_small, x, add, m);
#pragma unroll
              for (int z = 0; z < 4; ++z) {
                if (MASK && !((see[y] >> (e + z)) & 1u)) x[z] = m[z] = 0.f;
                w[y][e + z] = __float_as_uint(m[z]);
              }
              pk[e / 2] = pack2<F16>(x[0], x[1]);
              pk[e / 2 + 1] = pack2<F16>(x[2], x[3]);
            }
            tmem_st16(st + y * 16, pk);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.p_ready[y]);
          }
        };
        const bool small = CAP && cap_small(p, fmaxf(highest_abs(w[0]), highest_abs(w[1])), p.has_docs && kd < 0);
        if (__builtin_expect(masked, 0)) {
          if (CAP && small) phase(std::true_type{}, std::true_type{});
          else phase(std::true_type{}, std::false_type{});
        } else {
          if (CAP && small) phase(std::false_type{}, std::true_type{});
          else phase(std::false_type{}, std::false_type{});
        }

        float4 nd4[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) nd4[e] = lds_f4(stat + TILE * 4 + e * 16);
        ok = wait_for(sh.dp_full, it & 1, sh.abort_flag, 0x3303);
        if (!ok) break;
        tc_fence_after();
        auto gradients = [&](auto mask_tag) {
          constexpr bool MASK = decltype(mask_tag)::value;
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t d[32], pk[16];
            tmem_ld32(dp + y * 32, d);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 nd = nd4[y * 8 + e / 4];
              float a[4];
              f2_split(f2_mul(f2(w[y][e], w[y][e + 1]), f2_add(f2(d[e], d[e + 1]), f2(nd.x, nd.y))), a[0], a[1]);
              f2_split(f2_mul(f2(w[y][e + 2], w[y][e + 3]), f2_add(f2(d[e + 2], d[e + 3]), f2(nd.z, nd.w))), a[2], a[3]);
              if (MASK) {   // p is 0 there already, but dp of padding may be NaN
#pragma unroll
                for (int z = 0; z < 4; ++z)
                  if (!((see[y] >> (e + z)) & 1u)) a[z] = 0.f;
              }
              pk[e / 2] = pack2<F16>(a[0], a[1]);
              pk[e / 2 + 1] = pack2<F16>(a[2], a[3]);
            }
            tmem_st16(dp + y * 16, pk);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.ds_ready[y]);
          }
        };
        if (__builtin_expect(masked, 0)) gradients(std::true_type{});
        else gradients(std::false_type{});
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
          if (j < p.skv) write_row(o, out + x * 64, prm.wide != 0);
        }
      }
      tc_fence_before();   // the next unit's first products overwrite the accumulators
      unit_done(sh.sched, k);
    }
  }
  bwd_end(sh, tmem, p.err);
}

// Sums the splits of dk and dv, in order.  D / 4 lanes a row of one of the two.  Bound by its launch (2 x
// 96 keys of 8 heads: 5 us).
template <int D, bool F16>
__global__ void __launch_bounds__(256) dkv_join_kernel(const BwdParams prm) {
  wait_for_previous();
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

template <int D, bool F16, bool CAP, bool BIAS>
static int launch(const BwdParams& f, const CUtensorMap& q, const CUtensorMap& go, const CUtensorMap& k,
                  const CUtensorMap& v, cudaStream_t s) {
  using C = BwdCfg<D>;
  const Params& p = f.c;
  const auto kern = dkv_kernel<D, F16, CAP, BIAS>;
  int rc = prepare_kernel(reinterpret_cast<const void*>(kern), C::SMEM_BYTES);
  if (rc) return rc;
  const dim3 grid(unsigned(f.n_kt) * p.Hkv, p.bs, p.splits);
  rc = launch_kernel(kern, grid, kThreads, C::SMEM_BYTES, s, p.sq > 0 || p.has_docs, q, go, k, v, f);
  if (rc || p.splits == 1) return rc;
  const long long t = (long long)p.bs * p.Hkv * p.skv * 2 * (D / 4);
  return launch_kernel(dkv_join_kernel<D, F16>, dim3(unsigned((t + 255) / 256)), 256, 0, s, true, f);
}

int launch_dkv(const BwdParams& f, const CUtensorMap& q, const CUtensorMap& go, const CUtensorMap& k,
               const CUtensorMap& v, int d, bool f16, bool cap, cudaStream_t s) {
  const bool bias = f.c.slopes != nullptr;
#define ATTN_BWD_PICK(DD, FF)                                                                                   \
  if (d == DD && f16 == FF)                                                                                     \
    return cap ? (bias ? launch<DD, FF, true, true>(f, q, go, k, v, s) : launch<DD, FF, true, false>(f, q, go, k, v, s)) \
               : (bias ? launch<DD, FF, false, true>(f, q, go, k, v, s) : launch<DD, FF, false, false>(f, q, go, k, v, s));
  ATTN_BWD_PICK(128, false)
  ATTN_BWD_PICK(128, true)
  ATTN_BWD_PICK(64, false)
  ATTN_BWD_PICK(64, true)
#undef ATTN_BWD_PICK
  return ATTN_BWD_EUNSUPPORTED;
}

}  // namespace fused
}  // namespace attn_bwd
