// fused_common.cuh — what the fused attention kernels share: parameters, which keys a query
// sees, the list of key (or query) tiles a CTA visits, and the score transform.
//
// Scores are kept in units of log2: t = s * log2(e), so that p = 2^(t - t_max).
#pragma once
#include <cuda_fp16.h>

#include "fast_div.h"
#include "sm100.cuh"

namespace attn_bwd {
namespace fused {
using namespace sm100;

constexpr int TILE = 128;        // rows of a query tile, keys of a key tile
constexpr int kMaxList = 2048;   // documents: tiles of one unit at most
// Tiles of one unit at most: the scheduler and warps without rows wait for a whole unit, and waits give up
// after 2 s.  A capped tile takes up to 4 us, so a unit about 1 s.
constexpr int kMaxUnit = 1 << 18;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct DocRange;

struct Params {
  int bs, sq, skv, H, Hkv, G;
  int off;                 // position of query row 0: skv - sq
  int causal, has_docs;
  float scale;             // of the scores
  float scale_log2;        // scale * log2(e)
  float cap_u;             // softcap: scale / softcap (infinite where TanhSmall's coefficients are)
  float cap_in;            // 2 * log2(e) * scale / softcap
  float cap_out;           // softcap * log2(e)
  float cap_inv;           // 1 / cap_out
  float cap_poly[6];       // coefficients of TanhSmall
  const float* slopes;     // [H] or null
  const int* prefix;       // [bs] or null
  const int *qdoc, *kdoc;  // [bs, sq], [bs, skv] or null
  const DocRange *qrange, *krange;   // of the 128-position tiles, [bs, tiles]
  int n_tiles;             // tiles of the axis a CTA loops over
  int splits, tiles_per_split;
  FastDiv divG;            // heads of a group
  int* err;
};

// Bounded wait of a warp on an mbarrier phase, kept small in code: it occurs some twenty times a
// kernel, and the kernels' units are short enough for instruction fetches to count.  Gives up
// after kWaitLimitNs (or when another warp of the block has) and leaves its code in the block's
// flag, which report_error() passes on at the end.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* flag, int code) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P, Q;\n\t.reg .u64 t0, t1;\n\t.reg .u32 f;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2;\n\t"
      "@P bra DONE;\n\t"
      "mov.u64 t0, %%globaltimer;\n"
      "AGAIN:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2, %3;\n\t"
      "@P bra DONE;\n\t"
      "ld.volatile.shared.u32 f, [%4];\n\t"
      "setp.ne.u32 Q, f, 0;\n\t"
      "@Q bra DONE;\n\t"
      "mov.u64 t1, %%globaltimer;\n\t"
      "sub.u64 t1, t1, t0;\n\t"
      "setp.lt.u64 Q, t1, %5;\n\t"
      "@Q bra AGAIN;\n\t"
      "st.volatile.shared.u32 [%4], %6;\n"
      "DONE:\n\t"
      "selp.u32 %0, 1, 0, P;\n\t}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(kSuspendHintNs), "r"(smem_u32(const_cast<int*>(flag))), "l"(kWaitLimitNs),
        "r"(code)
      : "memory");
  return __all_sync(0xffffffffu, ok != 0);
}
// Barrier of some warps of one block, bounded like every wait (a named barrier would hold warps for
// good if one of them had given up): bar counts the warps, n their meetings so far.
__device__ __forceinline__ bool meet(uint64_t* bar, uint32_t& n, volatile int* flag, int code) {
  __syncwarp();
  if (lane_id() == 0) mbar_arrive(bar);
  return wait_for(bar, n++ & 1, flag, code);
}
__device__ __forceinline__ void report_error(volatile int* flag, int* err) {
  if (threadIdx.x == 0 && *flag) raise_error(err, *flag);
}

// The kernels of a call follow one another closely (programmatic dependent launch): each lets the next
// one's blocks in when its own blocks are on their last unit, and waits, after setting up barriers and
// TMEM and before it touches any tensor, for the one before it to have finished and its results to be
// visible.  Without such a launch neither does anything.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Number of keys (from key 0) that query row `r` of batch row b sees when documents are left
// out of account: a prefix, then causal.  Never above skv; 0 or less: none.
__device__ __forceinline__ int row_limit(const Params& p, int r, int pre) {
  if (!p.causal) return p.skv;
  return min(p.skv, max(r + p.off + 1, pre));
}

// Lowest and highest document number (>= 0) of some ids, and whether any id is negative.  No
// id >= 0: lo > hi.
struct DocRange {
  int lo, hi, neg, pad;
};
// The same on every lane of a warp.
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
  r.pad = 0;
  return r;
}
// Ranges of all key tiles, then (sq > 0) of all query tiles, one warp a tile: read once here instead of
// by every unit that looks at the tile (some 3 us, most of them the launch's).
static __global__ void __launch_bounds__(256) doc_ranges_kernel(const int* __restrict__ kdoc, int skv,
                                                                const int* __restrict__ qdoc, int sq, int bs,
                                                                DocRange* __restrict__ kr, DocRange* __restrict__ qr) {
  let_next_start();
  const int nk = (skv + TILE - 1) / TILE, nq = (sq + TILE - 1) / TILE;
  long long t = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const uint32_t lane = threadIdx.x & 31;
  const bool q = t >= (long long)bs * nk;
  if (q) t -= (long long)bs * nk;
  const int n = q ? nq : nk, s = q ? sq : skv;
  if (t >= (long long)bs * n) return;
  const int b = int(t / n), r0 = int(t - (long long)b * n) * TILE;
  const DocRange r = warp_doc_range((q ? qdoc : kdoc) + (size_t)b * s + r0, min(TILE, s - r0), lane);
  if (lane == 0) (q ? qr : kr)[t] = r;
}

// A tile of a CTA's loop: number (from the unit's first tile), whether single scores have to be
// masked, and whether rows of the streamed tile belong to no document and so are cleared before
// a product reads them.
constexpr uint32_t kEntMask = 0x8000u, kEntScrub = 0x4000u, kEntTile = 0x3fffu;
constexpr int kStSkip = 0, kStFull = 1, kStMask = 2;

// State of the pair (query range, key range): rows of the range [r0, r1], keys [j0, j1].
__device__ __forceinline__ int pair_state(const Params& p, int pre, int r0, int r1, int j0, int j1, const DocRange& qd,
                                          const DocRange& kd) {
  const int lim0 = row_limit(p, r0, pre), lim1 = row_limit(p, r1, pre);   // limits grow with the row
  if (lim1 <= j0 || qd.hi < qd.lo || kd.hi < kd.lo || qd.hi < kd.lo || kd.hi < qd.lo) return kStSkip;
  return lim0 > j1 && !qd.neg && !kd.neg && qd.lo == qd.hi && kd.lo == kd.hi ? kStFull : kStMask;
}

// Appends the lanes' tiles to a list, in order; one warp.  state: of tile t, kStSkip: left out.
__device__ __forceinline__ int list_append(uint16_t* list, int cnt, int t, int state, bool scrub, uint32_t lane) {
  const uint32_t vote = __ballot_sync(0xffffffffu, state != kStSkip);
  if (state != kStSkip)
    list[cnt + __popc(vote & ((1u << lane) - 1u))] =
        uint16_t(uint32_t(t) | (state == kStMask ? kEntMask : 0u) | (scrub ? kEntScrub : 0u));
  return cnt + __popc(vote);
}

// ---- units: a kernel's blocks are taken up by CTAs that stay, one an SM.  The scheduler warp
// asks the hardware for the next block that has not started (cluster launch control) while
// the current one is worked on, so its loads and first products start early and no SM waits
// for a launch.  Two slots: the unit in work and the next.
struct alignas(16) Unit {
  int x, y, z;     // block index; x < 0: no more units
  int n;           // documents: tiles of the list
};
struct Scheduler {
  Unit* slot;          // [2]
  uint64_t *full, *empty, *answer;
  uint64_t* ask;       // the producer has issued the last loads of a unit: time to take up another
  uint32_t handle;     // shared address of the hardware's answer (16 bytes)
};
__device__ __forceinline__ void ask_next(const Scheduler& s) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   s.handle),
               "r"(smem_u32(s.answer))
               : "memory");
}
// Block index of the answer; false: no block is left.
__device__ __forceinline__ bool read_answer(const Scheduler& s, int& x, int& y, int& z) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t"
      "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\t"
      "ld.shared.b128 h, [%4];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.u32 %3, 1, 0, p;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, %1, %2, _}, h;\n\t}\n"
      : "=&r"(x), "=&r"(y), "=&r"(z), "=&r"(ok)
      : "r"(s.handle)
      : "memory");
  return ok != 0;
}
// L2 prefetches for the unit that comes next, by the scheduler warp: its resident tiles are asked
// for only when this unit has done with their place.
__device__ __forceinline__ void prefetch_l2_4d(const CUtensorMap* m, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p) : "memory"); }

constexpr int kUnitReaders = 10;   // producer, tensor cores, 8 warps of rows
__device__ __forceinline__ void scheduler_init(const Scheduler& s) {
  for (int i = 0; i < 2; ++i) { mbar_init(&s.full[i], 1); mbar_init(&s.empty[i], kUnitReaders); }
  mbar_init(s.answer, 1);
  mbar_init(s.ask, 1);
}
// The scheduler warp.  build(unit, slot) -> n prepares a unit's list (one warp).
template <typename F>
__device__ __forceinline__ void run_scheduler(const Scheduler& s, volatile int* abort, int code, F build) {
  const uint32_t lane = lane_id();
  int x = blockIdx.x, y = blockIdx.y, z = blockIdx.z;
  bool have = true;
  for (uint32_t k = 0;; ++k) {
    const uint32_t i = k & 1;
    if (!wait_for(&s.empty[i], ((k >> 1) & 1) ^ 1, abort, code)) return;
    const int n = have ? build(x, y, z, i) : 0;
    __syncwarp();
    if (lane == 0) {
      s.slot[i] = Unit{have ? x : -1, y, z, n};
      mbar_arrive(&s.full[i]);
    }
    if (!have) {
      if (lane == 0) let_next_start();
      return;
    }
    // not earlier: a CTA that took its next unit at once would hold it while others run dry
    if (!wait_for(s.ask, k & 1, abort, code + 2)) return;
    if (lane == 0) {
      mbar_arrive_expect_tx(s.answer, 16);
      ask_next(s);
    }
    if (!wait_for(s.answer, k & 1, abort, code + 1)) return;
    have = read_answer(s, x, y, z);
    fence_proxy_async_smem();   // the next answer is written by the async proxy
    __syncwarp();
  }
}
// A reader's next unit; false: none left (or the kernel gives up).
__device__ __forceinline__ bool next_unit(const Scheduler& s, uint32_t k, Unit& u, volatile int* abort, int code) {
  if (!wait_for(&s.full[k & 1], (k >> 1) & 1, abort, code)) return false;
  u = s.slot[k & 1];
  return u.x >= 0;
}
__device__ __forceinline__ void ask_for_unit(const Scheduler& s) {   // producer
  __syncwarp();
  if (lane_id() == 0) mbar_arrive(s.ask);
}
__device__ __forceinline__ void unit_done(const Scheduler& s, uint32_t k) {
  __syncwarp();
  if (lane_id() == 0) mbar_arrive(&s.empty[k & 1]);
}

// ---- results: one row a lane, 32 values as 16 pairs, in two stores of 32 bytes (a whole sector
// each).  For rows that are no box of a tensor map: (position, head) rows, and keys' gradients in the
// caller's strides.  A store's address is a multiple of its width, and results need only 16-byte rows: wide
// (see wide_rows) says that all of them are multiples of 32.
__device__ __forceinline__ void write_row(const uint32_t (&w)[16], uint8_t* dst, bool wide) {
  if (__builtin_expect(wide, 1)) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + h * 32), "r"(w[8 * h]),
                   "r"(w[8 * h + 1]), "r"(w[8 * h + 2]), "r"(w[8 * h + 3]), "r"(w[8 * h + 4]), "r"(w[8 * h + 5]),
                   "r"(w[8 * h + 6]), "r"(w[8 * h + 7])
                   : "memory");
  } else {
#pragma unroll
    for (int h = 0; h < 4; ++h)
      *reinterpret_cast<uint4*>(dst + h * 16) = make_uint4(w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]);
  }
}

// The same through the warp's 2 KB of shared memory and one tensor store of 32 rows x 64 bytes (a map
// with a box of 32 x 32 and the 64-byte swizzle): the warp goes on while the rows leave.  Rows behind
// the end are cut off by the map.  (When it took write_row's place: 16 documents of 640, causal forward,
// 230 -> 203 us.)
__device__ __forceinline__ void store_rows(uint32_t stage, const CUtensorMap* m, const uint32_t (&w)[16], int c0, int c1,
                                           int c2, int c3, uint32_t lane) {
  if (lane == 0) bulk_wait_read0();   // the store before this one has read the place
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 4; ++c)
    sts128(stage + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4), make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]));
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(m)),
                 "r"(stage), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
                 : "memory");
    bulk_commit();
  }
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
__device__ __forceinline__ float4 lds_f4(uint32_t saddr) {
  const uint4 v = lds128(saddr);
  return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
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

// r = 1 / (1 + 2^z) of four z = 2 x log2(e): tanh x = 1 - 2r and tanh' x = 4 r (1 - r), both to
// fp32 accuracy.  Special functions bound the capped kernels, so four share one reciprocal,
// 1 / ((1 + a)(1 + b)(1 + c)(1 + d)); z is cut at 30 (r = 2^-30: the tanh is 1 in fp32) so that
// the product stays below 2^121.  fminf cuts a NaN to 30 as well, which keeps it from the other three;
// it is put back at the end (a minimum that passes NaN on and a sum with 0 x NaN instead took 2 % more of the
// capped, biased backward).
__device__ __forceinline__ void cap_r4(float (&z)[4]) {
  float a[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = 1.f + ex2(fminf(z[i], 30.f));
  const float ab = a[0] * a[1], cd = a[2] * a[3];
  const float inv = rcp(ab * cd);
  const float iab = inv * cd, icd = inv * ab;
  z[0] = z[0] != z[0] ? z[0] : iab * a[1];
  z[1] = z[1] != z[1] ? z[1] : iab * a[0];
  z[2] = z[2] != z[2] ? z[2] : icd * a[3];
  z[3] = z[3] != z[3] ? z[3] : icd * a[2];
}

// softcap tanh(scale x / softcap) log2(e) of raw scores with |scale x / softcap| <= 0.75: x (c0 + c1
// x^2 + ..), an odd polynomial fitted to the tanh by Remez exchange (largest relative error 3.7e-8)
// with both scales in its coefficients.  Capped layers rarely come near their cap, and this needs
// no special function: the warps of a tile whose scores all stay below take it.
constexpr float kTanhSmall = 0.75f;
constexpr double kTanhPoly[5] = {-0.3333306908607483, 0.13326521217823029, -0.0533902570605278, 0.019664913415908813,
                                 -0.0047694905661046505};
struct TanhSmall {
  uint64_t c[6];
  // kept in registers (a volatile move is not repeated where the constants are used)
  __device__ __forceinline__ explicit TanhSmall(const Params& p) {
#pragma unroll
    for (int i = 0; i < 6; ++i) asm volatile("mov.b64 %0, {%1, %1};" : "=l"(c[i]) : "f"(p.cap_poly[i]));
  }
  // the factor of x
  __device__ __forceinline__ uint64_t factor(uint64_t x) const {
    const uint64_t x2 = f2_mul(x, x);
    uint64_t y = f2_fma(c[5], x2, c[4]);
    y = f2_fma(y, x2, c[3]);
    y = f2_fma(y, x2, c[2]);
    y = f2_fma(y, x2, c[1]);
    return f2_fma(y, x2, c[0]);
  }
};
__device__ __forceinline__ float highest_abs(const uint32_t (&x)[32]) {
  float big = 0.f;
#pragma unroll
  for (int e = 0; e < 32; e += 2) big = fmaxf(big, fmaxf(fabsf(__uint_as_float(x[e])), fabsf(__uint_as_float(x[e + 1]))));
  return big;
}
// pad: this lane's row (or key) belongs to no document, so what it holds has no part in the choice.
__device__ __forceinline__ bool cap_small(const Params& p, float big, bool pad) {
  return __all_sync(0xffffffffu, pad || big * p.cap_u <= kTanhSmall);
}
// One raw score to softcap tanh(scale x / softcap) log2(e).  (Through the reciprocal alone a high
// cap would leave nothing of a low score.)
__device__ __forceinline__ float cap1(const Params& p, const TanhSmall& ts, float x) {
  float lo, hi;
  f2_split(f2_mul(ts.factor(f2(x, x)), f2(x, x)), lo, hi);
  return fabsf(x) * p.cap_u <= kTanhSmall ? lo : fmaf(-2.f * p.cap_out, rcp(1.f + ex2(x * p.cap_in)), p.cap_out);
}
// Four raw scores to softcap tanh(scale x / softcap) log2(e) + add.  SMALL: all below kTanhSmall.
template <bool SMALL>
__device__ __forceinline__ void cap4(const Params& p, const TanhSmall& ts, float (&x)[4], float add) {
  if (SMALL) {
    const uint64_t a2 = f2(add, add), v = f2(x[0], x[1]), w = f2(x[2], x[3]);
    f2_split(f2_fma(ts.factor(v), v, a2), x[0], x[1]);
    f2_split(f2_fma(ts.factor(w), w, a2), x[2], x[3]);
  } else {
    const float top = p.cap_out + add;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] *= p.cap_in;
    cap_r4(x);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = fmaf(-2.f * p.cap_out, x[i], top);
  }
}
// 32 of them, in place.
template <bool SMALL>
__device__ __forceinline__ void cap32(const Params& p, const TanhSmall& ts, uint32_t (&x)[32]) {
#pragma unroll
  for (int e = 0; e < 32; e += 4) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __uint_as_float(x[e + i]);
    cap4<SMALL>(p, ts, y, 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[e + i] = __float_as_uint(y[i]);
  }
}

// Which of 32 ids per word (this lane holds ids[k * 32 + lane] in v[k]) equal this lane's own id:
// one ballot a word for each different id of the warp's rows, usually one or two.
template <int N>
__device__ __forceinline__ void same_ids(const int (&v)[N], int id, uint32_t (&same)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) same[k] = 0u;
  uint32_t todo = __ballot_sync(0xffffffffu, id >= 0);
  while (todo) {
    const int cur = __shfl_sync(0xffffffffu, id, __ffs(int(todo)) - 1);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const uint32_t m = __ballot_sync(0xffffffffu, v[k] == cur);
      if (id == cur) same[k] = m;
    }
    todo &= ~__ballot_sync(0xffffffffu, id == cur);
  }
}
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

// kind::f16 instruction descriptor for fp16 (0) or bf16 (1) operands, f32 accumulator.
__host__ __device__ constexpr uint32_t idesc16(bool f16, int M, int N, bool a_mn, bool b_mn) {
  return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}
// The products below are called by a whole warp with `one` set in the lane that issues them (always
// the same one), not from a branch of that lane: descriptors then stay in uniform registers and are
// stepped by one addition, where a divergent branch moves each of them there and the issue of
// small products, not the tensor cores, sets the pace (backward of 4096 x 4096, 80 heads: 2750 us so,
// 2470 from uniform control flow).
__device__ __forceinline__ void umma_ss1(bool one, uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(uint32_t(one)));
}
// D[tmem] (+)= A[tmem] * B[smem]^T: A holds 16-bit pairs along K, one 32-bit column a pair.
__device__ __forceinline__ void umma_ts1(bool one, uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(uint32_t(one)));
}
__device__ __forceinline__ void commit1(bool one, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
      "r"(uint32_t(one))
      : "memory");
}
// Descriptor of a tile read along its rows (K-major), and of one read across them (MN-major).
// An offset of o bytes adds o / 16.
__device__ __forceinline__ uint64_t desc_k(uint32_t tile) { return sdesc_sw128(tile, 16, 1024); }
__device__ __forceinline__ uint64_t desc_mn(uint32_t tile) { return sdesc_sw128(tile, TILE * 128, 1024); }

// Product of a K-major A tile [128 x D] and a K-major B tile [128 x D] (or, with idesc for
// N = 64, its first 64 rows): D[128 x N].  Tiles are D / 64 blocks of [128 rows x 128 bytes],
// 128-byte swizzled.
template <int D>
__device__ __forceinline__ void mma_kk(bool one, uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const uint32_t o = ((kk >> 2) * (TILE * 128) + (kk & 3) * 32) >> 4;
    umma_ss1(one, d_tmem, a + o, b + o, idesc, kk > 0 ? 1u : 0u);
  }
}
// Product of A [128 x 128] in TMEM (columns a0.. for the first 64 of K, a1.. for the second) and a
// tile [128 rows x D] whose rows are K: D[128 x D] (+)=.  Steps [K0, K1) of 16 rows.
template <int D, int K0, int K1>
__device__ __forceinline__ void mma_tn(bool one, uint32_t d_tmem, uint32_t a0, uint32_t a1, uint64_t b, uint32_t idesc,
                                       bool accumulate) {
#pragma unroll
  for (int kk = K0; kk < K1; ++kk)
    umma_ts1(one, d_tmem, (kk < 4 ? a0 : a1) + (kk & 3) * 8, b + kk * (2048 >> 4), idesc, (accumulate || kk > 0) ? 1u : 0u);
}

// The steps of such a product whose A columns the weight warps hand over together: 32 of every
// thread's 64 columns (Y = 0 or 1).
template <int D, int Y>
__device__ __forceinline__ void mma_tn_part(bool one, uint32_t d_tmem, uint32_t a0, uint32_t a1, uint64_t b,
                                            uint32_t idesc, bool accumulate) {
  mma_tn<D, 2 * Y, 2 * Y + 2>(one, d_tmem, a0, a1, b, idesc, accumulate);
  mma_tn<D, 2 * Y + 4, 2 * Y + 6>(one, d_tmem, a0, a1, b, idesc, true);
}

// Clears the rows of a [128 x D] tile whose document is negative: the tensor cores would turn a NaN
// there times a probability of 0 into NaN.  (Rows behind the end arrive as zeros.)  One warp; the
// caller has waited for the tile and is the only one to read it.
template <int D>
__device__ __forceinline__ void scrub_rows(uint32_t tile, const int* ids, int n, uint32_t lane) {
  int id[TILE / 32];
#pragma unroll
  for (int k = 0; k < TILE / 32; ++k) {
    const int r = k * 32 + int(lane);
    id[k] = r < n ? __ldg(ids + r) : 0;
  }
#pragma unroll
  for (int k = 0; k < TILE / 32; ++k) {
    for (uint32_t bad = __ballot_sync(0xffffffffu, id[k] < 0); bad; bad &= bad - 1) {
      const int r = k * 32 + __ffs(int(bad)) - 1;
      if (int(lane) < D / 8) sts128(tile + (lane >> 3) * (TILE * 128) + r * 128 + (lane & 7) * 16, make_uint4(0, 0, 0, 0));
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
}

}  // namespace fused
}  // namespace attn_bwd
