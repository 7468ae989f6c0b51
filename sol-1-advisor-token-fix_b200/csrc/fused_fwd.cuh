// fused_fwd.cuh — attention forward: o = softmax(modified scores) v, with the row statistic
// lse = log(sum(exp(s))), in one pass over the keys (running maximum and sum).
//
// One CTA holds up to two query tiles of 128 rows and streams key / value tiles of 128 keys
// through a ring in shared memory; both tiles use each of them.  While the tensor cores work
// for one query tile, the other one's softmax runs:
//   warp 8  TMA producer      warp 9  tcgen05 issuer, TMEM owner
//   warps 0-3 softmax of tile 0, warps 4-7 of tile 1: one thread a row
// TMEM: two score tiles (128 columns each) and two outputs (D columns each).  The weights go
// back to TMEM as 16-bit pairs over the scores they came from and are the A operand of the
// second product, so they never touch shared memory.
//
// The running maximum lags: the accumulator is rescaled only where a row's maximum has grown by
// more than 2^8, so most tiles need no pass over it.  Weights are then at most 2^8 instead of
// 1, which neither fp32 sums nor 16-bit weights (relative rounding) notice.
//
// Rows of a query tile are 128 positions of one head or, where that needs fewer tiles, up to
// 128 (position, head) pairs of one group (few positions, as when tokens are generated): a
// group's heads read the same keys.
#pragma once
#include "fused_common.cuh"

namespace attn_bwd {
namespace fused {

struct FwdParams {
  Params c;
  int packed;          // rows are (position, head of the group) pairs
  int pos_per_tile;    // positions of a tile: 128, or 128 / G
  int pair_heads;      // unpacked: the two tiles are two heads of one group, else 256 positions
  int blocks_q;        // position blocks per (batch, head slot)
  int head_slots;      // units along the heads: kv heads, head pairs or heads
  void* o;             // [bs, sq, H, D]
  float* lse;          // [bs, H, sq]
  float* part_o;       // splits > 1: [split][bs * H * sq][D]
  float* part_lse;     // splits > 1: [split][bs * H * sq]
};

template <int D>
struct FwdCfg {
  static constexpr int TILE_BYTES = TILE * D * 2;
  static constexpr int ST = D == 128 ? 4 : 8;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_KV = 2 * TILE_BYTES;
  static constexpr int OFF_LIST = OFF_KV + ST * TILE_BYTES;
  static constexpr int OFF_STATE = OFF_LIST + kMaxList * 2;
  static constexpr int OFF_DOC = OFF_STATE + kMaxList;          // per softmax warp: 128 ids
  static constexpr int OFF_BAR = OFF_DOC + 8 * TILE * 4;
  static constexpr int NBAR = 1 + 2 * ST + 6;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int SMEM_BYTES = OFF_MISC + 64 + 1024;
  static_assert(SMEM_BYTES <= 227 * 1024, "forward kernel shared memory");
};

// Applies the score transform to 128 raw scores of one row (in place, log2 units).
// Keys j0..j0+127; lim: keys below it are seen; mask words: further keys taken out.
template <bool CAP>
__device__ __forceinline__ void transform_row(const Params& p, uint32_t (&s)[4][32], float slope2, float dist0) {
  const float sl = p.scale_log2;
#pragma unroll
  for (int g = 0; g < 4; ++g)
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      float x = __uint_as_float(s[g][i]);
      if (CAP) x = fmaf(-2.f * p.cap_out, cap_r(x * p.cap_in), p.cap_out);
      else x *= sl;
      x = fmaf(-slope2, fabsf(dist0 - float(g * 32 + i)), x);
      s[g][i] = __float_as_uint(x);
    }
}

template <int D, bool F16, bool CAP>
__global__ void __launch_bounds__(kThreads, 1)
fwd_kernel(const __grid_constant__ CUtensorMap tm_q,   // (d, h, s, b), box (64, heads of a row, positions, 1)
           const __grid_constant__ CUtensorMap tm_k,   // (d, s, h, b), box (64, 128, 1, 1)
           const __grid_constant__ CUtensorMap tm_v, const FwdParams prm) {
  using C = FwdCfg<D>;
  constexpr int ST = C::ST;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* q_full = bars;
  uint64_t* kv_full = bars + 1;
  uint64_t* kv_empty = kv_full + ST;
  uint64_t* s_full = kv_empty + ST;    // [2] scores ready
  uint64_t* p_ready = s_full + 2;      // [2] weights written
  uint64_t* o_done = p_ready + 2;      // [2] second product done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 4);
  int* n_list_slot = reinterpret_cast<int*>(smem + C::OFF_MISC + 8);
  uint16_t* list = reinterpret_cast<uint16_t*>(smem + C::OFF_LIST);
  uint8_t* states = smem + C::OFF_STATE;

  const Params& p = prm.c;
  const uint32_t warp = warp_id(), lane = lane_id();
  // unit: later positions see more keys and come first
  const int qb = prm.blocks_q - 1 - int(blockIdx.x) / prm.head_slots;
  const int slot = int(blockIdx.x) % prm.head_slots;
  const int b = blockIdx.y, split = blockIdx.z;
  const int ppt = prm.pos_per_tile;
  // tile t: first head, first position
  int kvh, head0, head1, pos0, pos1;
  if (prm.packed) {
    kvh = slot;
    head0 = head1 = kvh * p.G;
    pos0 = qb * 2 * ppt;
    pos1 = pos0 + ppt;
  } else if (prm.pair_heads) {
    head0 = slot * 2;
    head1 = head0 + 1;
    kvh = head0 / p.G;
    pos0 = pos1 = qb * TILE;
  } else {
    head0 = head1 = slot;
    kvh = head0 / p.G;
    pos0 = qb * 2 * TILE;
    pos1 = pos0 + TILE;
  }
  const int nt = pos1 < p.sq ? 2 : 1;
  const int last_pos = min(p.sq, (nt == 2 ? pos1 : pos0) + ppt) - 1;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < ST; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_ready[i], 4); mbar_init(&o_done[i], 1); }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 8 && lane == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  if (warp == 9) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }

  // key tiles of this CTA: [t0, t1) of the split, minus those that none of its rows sees
  const int t0 = split * p.tiles_per_split;
  const int t1 = min(p.n_tiles, t0 + p.tiles_per_split);
  const int pre = p.prefix ? __ldg(p.prefix + b) : 0;
  {
    DocRange qd{0, -1, false};
    if (p.has_docs) qd = warp_doc_range(p.qdoc + (size_t)b * p.sq + pos0, last_pos - pos0 + 1, lane);
    if (p.has_docs) {
      for (int t = t0 + int(warp); t < t1; t += kThreads / 32) {
        const int j0 = t * TILE, j1 = min(p.skv, j0 + TILE) - 1;
        const DocRange kd = warp_doc_range(p.kdoc + (size_t)b * p.skv + j0, j1 - j0 + 1, lane);
        // keys behind the end are masked like unseen ones
        int st = pair_state(p, pre, pos0, last_pos, j0, j0 + TILE - 1, true, qd, kd);
        if (st != kStSkip && kd.neg) st |= kStScrub;
        if (lane == 0) states[t - t0] = uint8_t(st);
      }
    } else {
      for (int t = t0 + int(threadIdx.x); t < t1; t += kThreads) {
        const int j0 = t * TILE;
        states[t - t0] = uint8_t(pair_state(p, pre, pos0, last_pos, j0, j0 + TILE - 1, false, qd, qd));
      }
    }
  }
  __syncthreads();
  if (warp == 0) {
    const int n = compact_list(states, max(0, t1 - t0), list, lane);
    if (lane == 0) *n_list_slot = n;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int n = *n_list_slot;
  int* err = p.err;

  if (warp >= 8) {
   regs_shrink();
   if (warp == 8) {
    // ---------------------------------------------------------------- producer
    if (n > 0) {
      if (lane == 0) {
        // a tile's box covers ppt positions x 1 head, or x the group's heads
        const int rows = prm.packed ? ppt * p.G : TILE;
        mbar_arrive_expect_tx(q_full, uint32_t(nt) * rows * D * 2);
        for (int t = 0; t < nt; ++t)
          for (int x = 0; x < D / 64; ++x)
            tma_load_4d(smem + C::OFF_Q + t * C::TILE_BYTES + x * (TILE * 128), &tm_q, q_full, x * 64,
                        t ? head1 : head0, t ? pos1 : pos0, b);
      }
      uint32_t si = 0;
      bool ok = true;
      for (int i = 0; i < n && ok; ++i) {
        const int j0 = (t0 + int(list[i] & kEntTile)) * TILE;
        for (int m = 0; m < 2; ++m) {
          const uint32_t s = si % ST;
          ok = warp_wait(&kv_empty[s], ((si / ST) & 1) ^ 1, abort_flag, err, 0x2101);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&kv_full[s], C::TILE_BYTES);
            for (int x = 0; x < D / 64; ++x)
              tma_load_4d(smem + C::OFF_KV + s * C::TILE_BYTES + x * (TILE * 128), m ? &tm_v : &tm_k, &kv_full[s],
                          x * 64, j0, kvh, b);
          }
          ++si;
        }
      }
      if (lane == 0) {
        mbar_drain(q_full, 0, err, 0x2111);
        for (uint32_t k = 0; k < uint32_t(ST) && k < si; ++k) {
          const uint32_t i = si - 1 - k;
          mbar_drain(&kv_full[i % ST], (i / ST) & 1, err, 0x2112);
        }
      }
      __syncwarp();
    }
   } else if (warp == 9) {
    // ---------------------------------------------------------------- tensor cores
    constexpr uint32_t id_s = idesc16(F16, TILE, TILE, false, false);
    constexpr uint32_t id_o = idesc16(F16, TILE, D, false, true);
    const uint32_t qs = smem_u32(smem + C::OFF_Q), kvs = smem_u32(smem + C::OFF_KV);
    auto stage = [&](uint32_t si) { return kvs + (si % ST) * C::TILE_BYTES; };
    auto full = [&](uint32_t si, int code) {
      return warp_wait(&kv_full[si % ST], (si / ST) & 1, abort_flag, err, code);
    };
    if (n > 0 && warp_wait(q_full, 0, abort_flag, err, 0x2201) && full(0, 0x2202)) {
      tc_fence_after();
      if (lane == 0) {
        for (int t = 0; t < nt; ++t) {
          mma_kk<D>(tmem + t * TILE, qs + t * C::TILE_BYTES, stage(0), id_s);
          umma_commit(&s_full[t]);
        }
        umma_commit(&kv_empty[0]);
      }
      __syncwarp();
      for (int i = 0; i < n; ++i) {
        const uint32_t kn = 2 * i + 2, vi = 2 * i + 1;
        if (!full(vi, 0x2203)) break;
        if (list[i] & kEntScrub) {
          const int j0 = (t0 + int(list[i] & kEntTile)) * TILE;
          scrub_rows<D>(stage(vi), p.kdoc + (size_t)b * p.skv + j0, p.skv - j0, lane);
        }
        if (i + 1 < n && !full(kn, 0x2204)) break;
        bool ok = true;
        for (int t = 0; t < nt && ok; ++t) {
          ok = warp_wait(&p_ready[t], i & 1, abort_flag, err, 0x2205);
          if (!ok) break;
          tc_fence_after();
          if (lane == 0) {
            mma_tn<D>(tmem + 2 * TILE + t * D, tmem + t * TILE, tmem + t * TILE + 32, stage(vi), id_o, i > 0);
            umma_commit(&o_done[t]);
            if (i + 1 < n) {   // after the last tile nobody waits for a free stage
              if (t == nt - 1) umma_commit(&kv_empty[vi % ST]);
              mma_kk<D>(tmem + t * TILE, qs + t * C::TILE_BYTES, stage(kn), id_s);
              umma_commit(&s_full[t]);
              if (t == nt - 1) umma_commit(&kv_empty[kn % ST]);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
      }
    }
   }
  } else {
    // ---------------------------------------------------------------- softmax, one thread a row
    regs_grow();
    const int t = warp >> 2;
    if (t < nt) {
      const int row = int(warp & 3) * 32 + int(lane);
      const uint32_t t_lane = uint32_t((warp & 3) * 32) << 16;
      const uint32_t t_s = tmem + t_lane + t * TILE, t_o = tmem + t_lane + 2 * TILE + t * D;
      int pos, head;
      bool valid;
      if (prm.packed) {
        const int r = row / p.G;
        pos = (t ? pos1 : pos0) + r;
        head = (t ? head1 : head0) + row - r * p.G;
        valid = r < ppt && pos < p.sq;
      } else {
        pos = (t ? pos1 : pos0) + row;
        head = t ? head1 : head0;
        valid = pos < p.sq;
      }
      int lim = valid ? row_limit(p, pos, pre) : 0;
      const int qd = (valid && p.has_docs) ? __ldg(p.qdoc + (size_t)b * p.sq + pos) : -1;
      if (p.has_docs && qd < 0) lim = 0;
      const bool any_valid = __any_sync(0xffffffffu, valid);   // warps of padding rows only pass barriers
      const float slope2 = (p.slopes && valid) ? __ldg(p.slopes + head) * kLog2e : 0.f;
      const bool raw = !CAP && !p.slopes;                      // raw scores scaled inside the exponent
      const float c = raw ? p.scale_log2 : 1.f;
      const float grow = 8.f / c;
      const int* kdoc = p.has_docs ? p.kdoc + (size_t)b * p.skv : nullptr;
      int* ids = reinterpret_cast<int*>(smem + C::OFF_DOC) + warp * TILE;

      float mref = -INFINITY;   // reference maximum (raw or log2 units)
      float l = 0.f;
      bool ok = true;
      for (int i = 0; i < n; ++i) {
        ok = warp_wait(&s_full[t], i & 1, abort_flag, err, 0x2301);
        if (!ok) break;
        tc_fence_after();
        if (any_valid) {
          const uint32_t ent = list[i];
          const int j0 = (t0 + int(ent & kEntTile)) * TILE;
          uint32_t s[4][32];
#pragma unroll
          for (int g = 0; g < 4; ++g) tmem_ld32(t_s + g * 32, s[g]);
          tmem_wait_ld();
          if (!raw) transform_row<CAP>(p, s, slope2, float(pos + p.off - j0));
          if (ent & kEntMask) {
            if (p.has_docs) {
              __syncwarp();
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int j = j0 + k * 32 + int(lane);
                ids[k * 32 + lane] = j < p.skv ? __ldg(kdoc + j) : -1;
              }
              __syncwarp();
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const int m = min(max(lim - j0 - g * 32, 0), 32);
              uint32_t see = m == 32 ? 0xffffffffu : (1u << m) - 1u;
              if (p.has_docs) {
                uint32_t same = 0;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                  const int4 d = *reinterpret_cast<const int4*>(ids + g * 32 + k * 4);
                  same |= (d.x == qd ? 1u : 0u) << (k * 4) | (d.y == qd ? 2u : 0u) << (k * 4) |
                          (d.z == qd ? 4u : 0u) << (k * 4) | (d.w == qd ? 8u : 0u) << (k * 4);
                }
                see &= same;
              }
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((see >> e) & 1u)) s[g][e] = 0xff800000u;   // -inf
            }
          }
          float mx[4];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float x = fmaxf(__uint_as_float(s[g][0]), __uint_as_float(s[g][1]));
#pragma unroll
            for (int e = 2; e < 32; e += 2) x = fmaxf(x, fmaxf(__uint_as_float(s[g][e]), __uint_as_float(s[g][e + 1])));
            mx[g] = x;
          }
          const float m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          if (__any_sync(0xffffffffu, m > mref + grow)) {
            const float mnew = fmaxf(mref, m);
            const float f = mref == mnew ? 1.f : ex2((mref - mnew) * c);   // 0 from a reference of -inf
            mref = mnew;
            l *= f;
            if (i > 0) {
              ok = warp_wait(&o_done[t], (i - 1) & 1, abort_flag, err, 0x2302);
              if (!ok) break;
              tc_fence_after();
#pragma unroll
              for (int x = 0; x < D / 32; ++x) {
                uint32_t o[2][16];
                tmem_ld16(t_o + x * 32, o[0]);
                tmem_ld16(t_o + x * 32 + 16, o[1]);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  o[0][e] = __float_as_uint(__uint_as_float(o[0][e]) * f);
                  o[1][e] = __float_as_uint(__uint_as_float(o[1][e]) * f);
                }
                tmem_st16(t_o + x * 32, o[0]);
                tmem_st16(t_o + x * 32 + 16, o[1]);
              }
            }
          }
          const float nm = mref == -INFINITY ? 0.f : -mref * c;
          const uint64_t c2 = f2(c, c), nm2 = f2(nm, nm);
          uint64_t sum0 = 0, sum1 = 0;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              float a0, a1, b0, b1;
              f2_split(f2_fma(f2(s[g][e], s[g][e + 1]), c2, nm2), a0, a1);
              f2_split(f2_fma(f2(s[g][e + 2], s[g][e + 3]), c2, nm2), b0, b1);
              a0 = ex2(a0); a1 = ex2(a1); b0 = ex2(b0); b1 = ex2(b1);
              sum0 = f2_add(sum0, f2(a0, a1));
              sum1 = f2_add(sum1, f2(b0, b1));
              w[e / 2] = pack2<F16>(a0, a1);
              w[e / 2 + 1] = pack2<F16>(b0, b1);
            }
            tmem_st16(t_s + g * 16, w);
          }
          float x0, x1, y0, y1;
          f2_split(sum0, x0, x1);
          f2_split(sum1, y0, y1);
          l += (x0 + x1) + (y0 + y1);
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[t]);
      }
      // ---- epilogue: o / l, and the row statistic
      if (ok && n > 0) ok = warp_wait(&o_done[t], (n - 1) & 1, abort_flag, err, 0x2303);
      if (ok && any_valid) {
        tc_fence_after();
        const bool empty = l == 0.f;
        const float inv = empty ? 0.f : 1.f / l;
        const float lse = empty ? -INFINITY : (mref * c + log2f(l)) * kLn2;
        const size_t rowi = ((size_t)b * p.H + head) * p.sq + pos;
        if (p.splits > 1) {
          const size_t ri = (size_t)split * p.bs * p.H * p.sq + rowi;
          if (valid) prm.part_lse[ri] = lse;
#pragma unroll
          for (int x = 0; x < D / 32; ++x) {
            uint32_t o[32];
            __syncwarp();
            if (n > 0) {
              tmem_ld32(t_o + x * 32, o);
              tmem_wait_ld();
            }
            if (valid) {
              float4* dst = reinterpret_cast<float4*>(prm.part_o + ri * D + x * 32);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                dst[e] = empty ? make_float4(0.f, 0.f, 0.f, 0.f)
                               : make_float4(__uint_as_float(o[4 * e]) * inv, __uint_as_float(o[4 * e + 1]) * inv,
                                             __uint_as_float(o[4 * e + 2]) * inv, __uint_as_float(o[4 * e + 3]) * inv);
            }
          }
        } else {
          if (valid) prm.lse[rowi] = lse;
          uint8_t* dst = static_cast<uint8_t*>(prm.o) + (((size_t)b * p.sq + pos) * p.H + head) * (D * 2);
#pragma unroll
          for (int x = 0; x < D / 32; ++x) {
            uint32_t o[32];
            __syncwarp();
            if (n > 0) {
              tmem_ld32(t_o + x * 32, o);
              tmem_wait_ld();
            }
            if (valid) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                uint32_t w[4];
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  w[y] = empty ? 0u : pack2<F16>(__uint_as_float(o[8 * e + 2 * y]) * inv,
                                                 __uint_as_float(o[8 * e + 2 * y + 1]) * inv);
                *reinterpret_cast<uint4*>(dst + x * 64 + e * 16) = make_uint4(w[0], w[1], w[2], w[3]);
              }
            }
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

// Joins the splits of every row: o = sum_s 2^(lse_s - lse) o_s.  One warp a row; the sum
// over splits runs in order, so equal inputs give equal bits.
template <int D, bool F16>
__global__ void __launch_bounds__(256) fwd_join_kernel(const FwdParams prm) {
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

}  // namespace fused
}  // namespace attn_bwd
