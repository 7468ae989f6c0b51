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
// In both, warp 8 is the TMA producer, warp 9 issues tcgen05, and warps 0-7 turn scores into
// weights: TMEM lane quadrant warp % 4, columns 64 * (warp / 4).. of each tile.
#pragma once
#include "fused_common.cuh"

namespace attn_bwd {
namespace fused {

constexpr int kMaxListBwd = 8192;   // tiles a backward CTA visits at most: 2^20 positions

struct BwdParams {
  Params c;
  int sq_pad;            // sq rounded up to tiles: row length of nlse and ndelta
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
  static constexpr int OFF_A = 0;                           // two resident tiles
  static constexpr int OFF_RING = 2 * TILE_BYTES;
  static constexpr int OFF_STAT = OFF_RING + ST * TILE_BYTES;   // dkv: 2 x (nlse, ndelta) of 128 rows
  static constexpr int OFF_DOC = OFF_STAT + 2 * 2 * TILE * 4;   // per warp: 64 ids
  static constexpr int OFF_LIST = OFF_DOC + 8 * 64 * 4;
  static constexpr int OFF_STATE = OFF_LIST + kMaxListBwd * 2;
  static constexpr int OFF_BAR = OFF_STATE + kMaxListBwd;
  static constexpr int NBAR = 1 + 2 * ST + 6;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int SMEM_BYTES = OFF_MISC + 64 + 1024;
  static_assert(SMEM_BYTES <= 227 * 1024, "backward kernel shared memory");
};

struct BwdShared {
  uint8_t* smem;
  uint64_t *res_full, *full, *empty, *s_full, *p_ready, *dp_full, *ds_ready, *done;
  uint32_t* tmem_slot;
  volatile int* abort_flag;
  int* n_list;
  uint16_t* list;
  uint8_t* states;
};
template <int D>
__device__ __forceinline__ BwdShared bwd_shared(uint8_t* raw) {
  using C = BwdCfg<D>;
  BwdShared s;
  s.smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint64_t* b = reinterpret_cast<uint64_t*>(s.smem + C::OFF_BAR);
  s.res_full = b;
  s.full = b + 1;
  s.empty = s.full + C::ST;
  s.s_full = s.empty + C::ST;
  s.p_ready = s.s_full + 2;   // dq: one s_full a score tile
  s.dp_full = s.p_ready + 1;
  s.ds_ready = s.dp_full + 1;
  s.done = s.ds_ready + 1;
  s.tmem_slot = reinterpret_cast<uint32_t*>(s.smem + C::OFF_MISC);
  s.abort_flag = reinterpret_cast<volatile int*>(s.smem + C::OFF_MISC + 4);
  s.n_list = reinterpret_cast<int*>(s.smem + C::OFF_MISC + 8);
  s.list = reinterpret_cast<uint16_t*>(s.smem + C::OFF_LIST);
  s.states = s.smem + C::OFF_STATE;
  return s;
}
__device__ __forceinline__ void bwd_init(const BwdShared& s, int st) {
  mbar_init(s.res_full, 1);
  for (int i = 0; i < st; ++i) { mbar_init(&s.full[i], 1); mbar_init(&s.empty[i], 1); }
  mbar_init(&s.s_full[0], 1);
  mbar_init(&s.s_full[1], 1);
  mbar_init(s.p_ready, 8);
  mbar_init(s.dp_full, 1);
  mbar_init(s.ds_ready, 8);
  mbar_init(s.done, 1);
  *s.abort_flag = 0;
  fence_barrier_init();
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

// Bits of 32 ids (shared memory) that equal `id`.
__device__ __forceinline__ uint32_t same_bits(const int* ids, int id) {
  uint32_t same = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int4 d = *reinterpret_cast<const int4*>(ids + k * 4);
    same |= (d.x == id ? 1u : 0u) << (k * 4) | (d.y == id ? 2u : 0u) << (k * 4) | (d.z == id ? 4u : 0u) << (k * 4) |
            (d.w == id ? 8u : 0u) << (k * 4);
  }
  return same;
}
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

// One weight from a raw score; w receives what ds is multiplied by: p, or p tanh'.
template <bool CAP>
__device__ __forceinline__ float weight(const Params& p, float x, float bias, float nlse, float& w) {
  if (CAP) {
    const float r = cap_r(x * p.cap_in);
    const float e = ex2(fmaf(-2.f * p.cap_out, r, p.cap_out) + bias + nlse);
    w = e * (4.f * r * (1.f - r));
    return e;
  }
  w = ex2(fmaf(x, p.scale_log2, bias + nlse));
  return w;
}

// ------------------------------------------------------------------------------- dk, dv
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
  // unit: earlier keys are seen by more queries and come first
  const int jt = int(blockIdx.x) / p.Hkv, kvh = int(blockIdx.x) % p.Hkv;
  const int b = blockIdx.y, split = blockIdx.z;
  const int j0 = jt * TILE;
  if (threadIdx.x == 0) bwd_init(sh, ST);
  if (warp == 8 && lane == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_do);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  if (warp == 9) { tmem_alloc(sh.tmem_slot, 512); tmem_relinquish(); }
  const int pre = p.prefix ? __ldg(p.prefix + b) : 0;
  {
    const int j1 = min(p.skv, j0 + TILE) - 1;
    if (p.has_docs) {
      const DocRange kd = warp_doc_range(p.kdoc + (size_t)b * p.skv + j0, j1 - j0 + 1, lane);
      for (int t = int(warp); t < p.n_tiles; t += kThreads / 32) {
        const int r0 = t * TILE, r1 = min(p.sq, r0 + TILE) - 1;
        const DocRange qd = warp_doc_range(p.qdoc + (size_t)b * p.sq + r0, r1 - r0 + 1, lane);
        int st = pair_state(p, pre, r0, r1, j0, j1, true, qd, kd);
        if (st != kStSkip && qd.neg) st |= kStScrub;
        if (lane == 0) sh.states[t] = uint8_t(st);
      }
    } else {
      const DocRange none{0, -1, false};
      for (int t = int(threadIdx.x); t < p.n_tiles; t += kThreads) {
        const int r0 = t * TILE, r1 = min(p.sq, r0 + TILE) - 1;
        sh.states[t] = uint8_t(pair_state(p, pre, r0, r1, j0, j1, false, none, none));
      }
    }
  }
  __syncthreads();
  if (warp == 0) {
    const int cnt = compact_list(sh.states, p.n_tiles, sh.list, lane);
    if (lane == 0) *sh.n_list = cnt;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *sh.tmem_slot;
  const int nl = *sh.n_list;
  // items of this CTA: (head of the group, listed tile) pairs [i0, i1)
  const int items = nl * p.G;
  const int per = (items + p.splits - 1) / p.splits;
  const int i0 = min(items, split * per), n = min(items, i0 + per) - i0;
  int* err = p.err;
  const uint32_t t_st = tmem, t_dp = tmem + TILE, t_dv = tmem + 2 * TILE, t_dk = t_dv + D;

  if (warp >= 8) {
    regs_shrink();
    if (warp == 8) {
      // -------------------------------------------------------------- producer
      if (n > 0) {
        if (lane == 0) {
          mbar_arrive_expect_tx(sh.res_full, 2 * C::TILE_BYTES);
          for (int m = 0; m < 2; ++m)
            for (int x = 0; x < D / 64; ++x)
              tma_load_4d(sh.smem + C::OFF_A + m * C::TILE_BYTES + x * (TILE * 128), m ? &tm_v : &tm_k, sh.res_full,
                          x * 64, j0, kvh, b);
        }
        uint32_t si = 0;
        bool ok = true;
        int g = i0 / nl, t = i0 - g * nl;
        for (int i = 0; i < n && ok; ++i) {
          const int r0 = int(sh.list[t] & kEntTile) * TILE, h = kvh * p.G + g;
          for (int m = 0; m < 2; ++m) {
            const uint32_t s = si % ST;
            ok = warp_wait(&sh.empty[s], ((si / ST) & 1) ^ 1, sh.abort_flag, err, 0x3101);
            if (!ok) break;
            if (lane == 0) {
              mbar_arrive_expect_tx(&sh.full[s], C::TILE_BYTES + (m ? 0 : 2 * TILE * 4));
              for (int x = 0; x < D / 64; ++x)
                tma_load_4d(sh.smem + C::OFF_RING + s * C::TILE_BYTES + x * (TILE * 128), m ? &tm_do : &tm_q,
                            &sh.full[s], x * 64, r0, h, b);
              if (!m) {   // the rows' statistics arrive with the queries
                const size_t at = ((size_t)b * p.H + h) * prm.sq_pad + r0;
                uint8_t* dst = sh.smem + C::OFF_STAT + (i & 1) * (2 * TILE * 4);
                bulk_load(dst, prm.nlse + at, TILE * 4, &sh.full[s]);
                bulk_load(dst + TILE * 4, prm.ndelta + at, TILE * 4, &sh.full[s]);
              }
            }
            ++si;
          }
          if (++t == nl) { t = 0; ++g; }
        }
        if (lane == 0) {
          mbar_drain(sh.res_full, 0, err, 0x3111);
          for (uint32_t k = 0; k < uint32_t(ST) && k < si; ++k) {
            const uint32_t i = si - 1 - k;
            mbar_drain(&sh.full[i % ST], (i / ST) & 1, err, 0x3112);
          }
        }
        __syncwarp();
      }
    } else if (warp == 9) {
      // -------------------------------------------------------------- tensor cores
      constexpr uint32_t id_s = idesc16(F16, TILE, TILE, false, false);
      constexpr uint32_t id_g = idesc16(F16, TILE, D, false, true);
      const uint32_t ks = smem_u32(sh.smem + C::OFF_A), vs = ks + C::TILE_BYTES;
      const uint32_t ring = smem_u32(sh.smem + C::OFF_RING);
      auto stage = [&](int si) { return ring + (uint32_t(si) % ST) * C::TILE_BYTES; };
      int t = n > 0 ? i0 % nl : 0;
      // waits for slot si (and clears rows of padding: their products with 0 must be 0)
      auto arrived = [&](int si, int tt, int code) {
        if (!warp_wait(&sh.full[uint32_t(si) % ST], (uint32_t(si) / ST) & 1, sh.abort_flag, err, code)) return false;
        if (sh.list[tt] & kEntScrub) {
          const int r0 = int(sh.list[tt] & kEntTile) * TILE;
          scrub_rows<D>(stage(si), p.qdoc + (size_t)b * p.sq + r0, p.sq - r0, lane);
        }
        return true;
      };
      if (n > 0 && warp_wait(sh.res_full, 0, sh.abort_flag, err, 0x3201) && arrived(0, t, 0x3202) &&
          arrived(1, t, 0x3203)) {
        tc_fence_after();
        if (lane == 0) {
          mma_kk<D>(t_st, ks, stage(0), id_s);
          umma_commit(sh.s_full);
          mma_kk<D>(t_dp, vs, stage(1), id_s);
          umma_commit(sh.dp_full);
        }
        __syncwarp();
        for (int i = 0; i < n; ++i) {
          const bool more = i + 1 < n;
          if (++t == nl) t = 0;
          if (more && !arrived(2 * i + 2, t, 0x3204)) break;
          if (!warp_wait(sh.p_ready, i & 1, sh.abort_flag, err, 0x3205)) break;
          tc_fence_after();
          if (lane == 0) {
            mma_tn<D>(t_dv, t_st, t_st + 64, stage(2 * i + 1), id_g, i > 0);
            if (i + 2 < n) umma_commit(&sh.empty[(2 * i + 1) % ST]);
            if (more) {
              mma_kk<D>(t_st, ks, stage(2 * i + 2), id_s);
              umma_commit(sh.s_full);
            }
          }
          __syncwarp();
          if (more && !arrived(2 * i + 3, t, 0x3206)) break;
          if (!warp_wait(sh.ds_ready, i & 1, sh.abort_flag, err, 0x3207)) break;
          tc_fence_after();
          if (lane == 0) {
            mma_tn<D>(t_dk, t_dp, t_dp + 64, stage(2 * i), id_g, i > 0);
            if (i + 2 < n) umma_commit(&sh.empty[(2 * i) % ST]);
            if (more) {
              mma_kk<D>(t_dp, vs, stage(2 * i + 3), id_s);
              umma_commit(sh.dp_full);
            } else {
              umma_commit(sh.done);
            }
          }
          __syncwarp();
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- weights: one key a thread, 64 queries
    regs_grow();
    const int half = int(warp) >> 2, j = j0 + int(warp & 3) * 32 + int(lane);
    const uint32_t t_lane = uint32_t((warp & 3) * 32) << 16;
    const uint32_t st = t_st + t_lane + half * 64, dp = t_dp + t_lane + half * 64;
    const int kd = (p.has_docs && j < p.skv) ? __ldg(p.kdoc + (size_t)b * p.skv + j) : -1;
    int* ids = reinterpret_cast<int*>(sh.smem + C::OFF_DOC) + warp * 64;
    const bool plain = !CAP && !p.slopes;
    const uint64_t c2 = f2(p.scale_log2, p.scale_log2);
    bool ok = true;
    int g = n > 0 ? i0 / nl : 0, t = n > 0 ? i0 - g * nl : 0;
    for (int i = 0; i < n; ++i) {
      const uint32_t ent = sh.list[t];
      const int r0 = int(ent & kEntTile) * TILE + half * 64;   // first of this thread's query rows
      const float* stat = reinterpret_cast<const float*>(sh.smem + C::OFF_STAT + (i & 1) * (2 * TILE * 4)) + half * 64;
      uint32_t see[2] = {0xffffffffu, 0xffffffffu};
      if (ent & kEntMask) {
        if (p.has_docs) {
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int r = r0 + k * 32 + int(lane);
            ids[k * 32 + lane] = r < p.sq ? __ldg(p.qdoc + (size_t)b * p.sq + r) : -1;
          }
          __syncwarp();
        }
        // seen by row r if j < prefix or j <= r + off: rows from j - off on
        const int first = (!p.causal || j < pre) ? 0 : j - p.off - r0;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          see[k] = ~low_bits(first - k * 32);
          if (p.has_docs) see[k] = kd < 0 ? 0u : see[k] & same_bits(ids + k * 32, kd);
        }
      }
      ok = warp_wait(sh.s_full, i & 1, sh.abort_flag, err, 0x3301) &&
           warp_wait(&sh.full[(2 * i) % ST], ((2 * i) / ST) & 1, sh.abort_flag, err, 0x3302);
      if (!ok) break;
      tc_fence_after();
      uint32_t w[2][32];   // scores, then what ds is multiplied by
#pragma unroll
      for (int k = 0; k < 2; ++k) tmem_ld32(st + k * 32, w[k]);
      tmem_wait_ld();
      const float slope2 = p.slopes ? __ldg(p.slopes + kvh * p.G + g) * kLog2e : 0.f;
      const float dist0 = float(r0 + p.off - j);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 nl4 = *reinterpret_cast<const float4*>(stat + k * 32 + e);
          float a[4];
          if (plain) {
            f2_split(f2_fma(f2(w[k][e], w[k][e + 1]), c2, f2(nl4.x, nl4.y)), a[0], a[1]);
            f2_split(f2_fma(f2(w[k][e + 2], w[k][e + 3]), c2, f2(nl4.z, nl4.w)), a[2], a[3]);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              a[y] = ex2(a[y]);
              if (!((see[k] >> (e + y)) & 1u)) a[y] = 0.f;
              w[k][e + y] = __float_as_uint(a[y]);
            }
          } else {
            const float nls[4] = {nl4.x, nl4.y, nl4.z, nl4.w};
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              float m;
              a[y] = weight<CAP>(p, __uint_as_float(w[k][e + y]), -slope2 * fabsf(dist0 + float(k * 32 + e + y)),
                                 nls[y], m);
              if (!((see[k] >> (e + y)) & 1u)) a[y] = m = 0.f;
              w[k][e + y] = __float_as_uint(m);
            }
          }
          pk[e / 2] = pack2<F16>(a[0], a[1]);
          pk[e / 2 + 1] = pack2<F16>(a[2], a[3]);
        }
        tmem_st16(st + k * 16, pk);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sh.p_ready);

      ok = warp_wait(sh.dp_full, i & 1, sh.abort_flag, err, 0x3303);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t d[32], pk[16];
        tmem_ld32(dp + k * 32, d);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 nd = *reinterpret_cast<const float4*>(stat + TILE + k * 32 + e);
          float a[4];
          f2_split(f2_mul(f2(w[k][e], w[k][e + 1]), f2_add(f2(d[e], d[e + 1]), f2(nd.x, nd.y))), a[0], a[1]);
          f2_split(f2_mul(f2(w[k][e + 2], w[k][e + 3]), f2_add(f2(d[e + 2], d[e + 3]), f2(nd.z, nd.w))), a[2], a[3]);
          if (ent & kEntMask) {
#pragma unroll
            for (int y = 0; y < 4; ++y)
              if (!((see[k] >> (e + y)) & 1u)) a[y] = 0.f;
          }
          pk[e / 2] = pack2<F16>(a[0], a[1]);
          pk[e / 2 + 1] = pack2<F16>(a[2], a[3]);
        }
        tmem_st16(dp + k * 16, pk);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sh.ds_ready);
      if (++t == nl) { t = 0; ++g; }
    }
    // ---- epilogue: warps 0-3 write dv, warps 4-7 dk
    if (ok && n > 0) ok = warp_wait(sh.done, 0, sh.abort_flag, err, 0x3304);
    if (ok) {
      tc_fence_after();
      const float f = half ? p.scale : 1.f;
      const uint32_t src = (half ? t_dk : t_dv) + t_lane;
      uint8_t* out = half ? static_cast<uint8_t*>(prm.dk) + 2 * (b * prm.dks[0] + kvh * prm.dks[1] + j * prm.dks[2])
                          : static_cast<uint8_t*>(prm.dv) + 2 * (b * prm.dvs[0] + kvh * prm.dvs[1] + j * prm.dvs[2]);
      float* part = p.splits > 1
          ? prm.part + (((((size_t)split * p.bs + b) * p.Hkv + kvh) * p.skv + j) * 2 + (half ? 0 : 1)) * D : nullptr;
#pragma unroll
      for (int x = 0; x < D / 32; ++x) {
        uint32_t v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = 0u;
        __syncwarp();
        if (n > 0) {
          tmem_ld32(src + x * 32, v);
          tmem_wait_ld();
        }
        if (j >= p.skv) continue;
        if (p.splits > 1) {
          float4* dst = reinterpret_cast<float4*>(part + x * 32);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            dst[e] = make_float4(__uint_as_float(v[4 * e]) * f, __uint_as_float(v[4 * e + 1]) * f,
                                 __uint_as_float(v[4 * e + 2]) * f, __uint_as_float(v[4 * e + 3]) * f);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t o[4];
#pragma unroll
            for (int y = 0; y < 4; ++y)
              o[y] = pack2<F16>(__uint_as_float(v[8 * e + 2 * y]) * f, __uint_as_float(v[8 * e + 2 * y + 1]) * f);
            *reinterpret_cast<uint4*>(out + x * 64 + e * 16) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
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
  const int nqt = (p.sq + TILE - 1) / TILE;
  const int qt = nqt - 1 - int(blockIdx.x) / p.H, h = int(blockIdx.x) % p.H;   // later queries see more: first
  const int b = blockIdx.y, kvh = h / p.G;
  const int r0 = qt * TILE, r1 = min(p.sq, r0 + TILE) - 1;
  if (threadIdx.x == 0) bwd_init(sh, ST);
  if (warp == 8 && lane == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_do);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  if (warp == 9) { tmem_alloc(sh.tmem_slot, 512); tmem_relinquish(); }
  const int pre = p.prefix ? __ldg(p.prefix + b) : 0;
  const int n_kt = (p.skv + TILE - 1) / TILE;
  if (p.has_docs) {
    const DocRange qd = warp_doc_range(p.qdoc + (size_t)b * p.sq + r0, r1 - r0 + 1, lane);
    for (int t = int(warp); t < n_kt; t += kThreads / 32) {
      const int j0 = t * TILE, j1 = min(p.skv, j0 + TILE) - 1;
      const DocRange kd = warp_doc_range(p.kdoc + (size_t)b * p.skv + j0, j1 - j0 + 1, lane);
      int st = pair_state(p, pre, r0, r1, j0, j0 + TILE - 1, true, qd, kd);
      if (st != kStSkip && kd.neg) st |= kStScrub;
      if (lane == 0) sh.states[t] = uint8_t(st);
    }
  } else {
    const DocRange none{0, -1, false};
    for (int t = int(threadIdx.x); t < n_kt; t += kThreads)
      sh.states[t] = uint8_t(pair_state(p, pre, r0, r1, t * TILE, t * TILE + TILE - 1, false, none, none));
  }
  __syncthreads();
  if (warp == 0) {
    const int cnt = compact_list(sh.states, n_kt, sh.list, lane);
    if (lane == 0) *sh.n_list = cnt;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *sh.tmem_slot;
  const int n = *sh.n_list;
  int* err = p.err;
  const uint32_t t_dp = tmem + 2 * TILE, t_dq = tmem + 3 * TILE;

  if (warp >= 8) {
    regs_shrink();
    if (warp == 8) {
      // -------------------------------------------------------------- producer
      if (n > 0) {
        if (lane == 0) {
          mbar_arrive_expect_tx(sh.res_full, 2 * C::TILE_BYTES);
          for (int m = 0; m < 2; ++m)
            for (int x = 0; x < D / 64; ++x)
              tma_load_4d(sh.smem + C::OFF_A + m * C::TILE_BYTES + x * (TILE * 128), m ? &tm_do : &tm_q, sh.res_full,
                          x * 64, r0, h, b);
        }
        uint32_t si = 0;
        bool ok = true;
        for (int i = 0; i < n && ok; ++i) {
          const int j0 = int(sh.list[i] & kEntTile) * TILE;
          for (int m = 0; m < 2; ++m) {
            const uint32_t s = si % ST;
            ok = warp_wait(&sh.empty[s], ((si / ST) & 1) ^ 1, sh.abort_flag, err, 0x4101);
            if (!ok) break;
            if (lane == 0) {
              mbar_arrive_expect_tx(&sh.full[s], C::TILE_BYTES);
              for (int x = 0; x < D / 64; ++x)
                tma_load_4d(sh.smem + C::OFF_RING + s * C::TILE_BYTES + x * (TILE * 128), m ? &tm_v : &tm_k,
                            &sh.full[s], x * 64, j0, kvh, b);
            }
            ++si;
          }
        }
        if (lane == 0) {
          mbar_drain(sh.res_full, 0, err, 0x4111);
          for (uint32_t k = 0; k < uint32_t(ST) && k < si; ++k) {
            const uint32_t i = si - 1 - k;
            mbar_drain(&sh.full[i % ST], (i / ST) & 1, err, 0x4112);
          }
        }
        __syncwarp();
      }
    } else if (warp == 9) {
      // -------------------------------------------------------------- tensor cores
      constexpr uint32_t id_s = idesc16(F16, TILE, TILE, false, false);
      constexpr uint32_t id_g = idesc16(F16, TILE, D, false, true);
      const uint32_t qs = smem_u32(sh.smem + C::OFF_A), dos = qs + C::TILE_BYTES;
      const uint32_t ring = smem_u32(sh.smem + C::OFF_RING);
      auto stage = [&](int si) { return ring + (uint32_t(si) % ST) * C::TILE_BYTES; };
      auto arrived = [&](int si, int code) {
        if (!warp_wait(&sh.full[uint32_t(si) % ST], (uint32_t(si) / ST) & 1, sh.abort_flag, err, code)) return false;
        const uint32_t ent = sh.list[si >> 1];
        if (!(si & 1) && (ent & kEntScrub)) {
          const int j0 = int(ent & kEntTile) * TILE;
          scrub_rows<D>(stage(si), p.kdoc + (size_t)b * p.skv + j0, p.skv - j0, lane);
        }
        return true;
      };
      if (n > 0 && warp_wait(sh.res_full, 0, sh.abort_flag, err, 0x4201) && arrived(0, 0x4202) && arrived(1, 0x4203) &&
          (n < 2 || arrived(2, 0x4204))) {
        tc_fence_after();
        if (lane == 0) {
          mma_kk<D>(tmem, qs, stage(0), id_s);
          umma_commit(&sh.s_full[0]);
          mma_kk<D>(t_dp, dos, stage(1), id_s);
          umma_commit(sh.dp_full);
          if (n > 2) umma_commit(&sh.empty[1 % ST]);
          if (n > 1) {
            mma_kk<D>(tmem + TILE, qs, stage(2), id_s);
            umma_commit(&sh.s_full[1]);
          }
        }
        __syncwarp();
        for (int i = 0; i < n; ++i) {
          if (i + 1 < n && !arrived(2 * i + 3, 0x4205)) break;
          if (!warp_wait(sh.ds_ready, i & 1, sh.abort_flag, err, 0x4206)) break;
          tc_fence_after();
          const uint32_t t_s = tmem + (i & 1) * TILE;
          if (lane == 0) {
            if (i + 1 < n) {
              mma_kk<D>(t_dp, dos, stage(2 * i + 3), id_s);
              umma_commit(sh.dp_full);
              if (i + 3 < n) umma_commit(&sh.empty[(2 * i + 3) % ST]);
            }
            mma_tn<D>(t_dq, t_s, t_s + 64, stage(2 * i), id_g, i > 0);
            if (i + 2 < n) umma_commit(&sh.empty[(2 * i) % ST]);
            if (i + 1 == n) umma_commit(sh.done);
          }
          __syncwarp();
          if (i + 2 < n) {
            if (!arrived(2 * i + 4, 0x4207)) break;
            tc_fence_after();
            if (lane == 0) {
              mma_kk<D>(t_s, qs, stage(2 * i + 4), id_s);
              umma_commit(&sh.s_full[i & 1]);
            }
            __syncwarp();
          }
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- weights: one query a thread, 64 keys
    regs_grow();
    const int half = int(warp) >> 2, row = r0 + int(warp & 3) * 32 + int(lane);
    const uint32_t t_lane = uint32_t((warp & 3) * 32) << 16;
    const bool valid = row < p.sq;
    const size_t ri = ((size_t)b * p.H + h) * prm.sq_pad + row;
    const float nlse = prm.nlse[ri], nd = prm.ndelta[ri];   // padded to whole tiles
    const int lim = valid ? row_limit(p, row, pre) : 0;
    const int qd = (valid && p.has_docs) ? __ldg(p.qdoc + (size_t)b * p.sq + row) : -1;
    const float slope2 = p.slopes ? __ldg(p.slopes + h) * kLog2e : 0.f;
    int* ids = reinterpret_cast<int*>(sh.smem + C::OFF_DOC) + warp * 64;
    const bool plain = !CAP && !p.slopes;
    const uint64_t c2 = f2(p.scale_log2, p.scale_log2), nl2 = f2(nlse, nlse), nd2 = f2(nd, nd);
    const uint32_t dp = t_dp + t_lane + half * 64;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const uint32_t ent = sh.list[i];
      const int j0 = int(ent & kEntTile) * TILE + half * 64;
      const uint32_t st = tmem + (i & 1) * TILE + t_lane + half * 64;
      uint32_t see[2] = {0xffffffffu, 0xffffffffu};
      if (ent & kEntMask) {
        if (p.has_docs) {
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int j = j0 + k * 32 + int(lane);
            ids[k * 32 + lane] = j < p.skv ? __ldg(p.kdoc + (size_t)b * p.skv + j) : -1;
          }
          __syncwarp();
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          see[k] = low_bits(lim - j0 - k * 32);
          if (p.has_docs) see[k] = qd < 0 ? 0u : see[k] & same_bits(ids + k * 32, qd);
        }
      }
      ok = warp_wait(&sh.s_full[i & 1], (i >> 1) & 1, sh.abort_flag, err, 0x4301);
      if (!ok) break;
      tc_fence_after();
      uint32_t w[2][32];
#pragma unroll
      for (int k = 0; k < 2; ++k) tmem_ld32(st + k * 32, w[k]);
      tmem_wait_ld();
      const float dist0 = float(row + p.off - j0);
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          if (plain) {
            float a0, a1;
            f2_split(f2_fma(f2(w[k][e], w[k][e + 1]), c2, nl2), a0, a1);
            w[k][e] = __float_as_uint(ex2(a0));
            w[k][e + 1] = __float_as_uint(ex2(a1));
          } else {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              float m;
              weight<CAP>(p, __uint_as_float(w[k][e + y]), -slope2 * fabsf(dist0 - float(k * 32 + e + y)), nlse, m);
              w[k][e + y] = __float_as_uint(m);
            }
          }
        }
      ok = warp_wait(sh.dp_full, i & 1, sh.abort_flag, err, 0x4302);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t d[32], pk[16];
        tmem_ld32(dp + k * 32, d);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float a0, a1;
          f2_split(f2_mul(f2(w[k][e], w[k][e + 1]), f2_add(f2(d[e], d[e + 1]), nd2)), a0, a1);
          if (ent & kEntMask) {
            if (!((see[k] >> e) & 1u)) a0 = 0.f;
            if (!((see[k] >> (e + 1)) & 1u)) a1 = 0.f;
          }
          pk[e / 2] = pack2<F16>(a0, a1);
        }
        tmem_st16(st + k * 16, pk);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sh.ds_ready);
    }
    // ---- epilogue: each half of the warps writes half of the columns
    if (ok && n > 0) ok = warp_wait(sh.done, 0, sh.abort_flag, err, 0x4303);
    if (ok) {
      tc_fence_after();
      uint8_t* out = static_cast<uint8_t*>(prm.dq) + 2 * (b * prm.dqs[0] + h * prm.dqs[1] + row * prm.dqs[2]) +
                     half * D;
#pragma unroll
      for (int x = 0; x < D / 64; ++x) {
        uint32_t v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = 0u;
        __syncwarp();
        if (n > 0) {
          tmem_ld32(t_dq + t_lane + half * (D / 2) + x * 32, v);
          tmem_wait_ld();
        }
        if (!valid) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t o[4];
#pragma unroll
          for (int y = 0; y < 4; ++y)
            o[y] = pack2<F16>(__uint_as_float(v[8 * e + 2 * y]) * p.scale, __uint_as_float(v[8 * e + 2 * y + 1]) * p.scale);
          *reinterpret_cast<uint4*>(out + x * 64 + e * 16) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace fused
}  // namespace attn_bwd
