// rope.cu — rotary positions of queries and keys (and of their gradients) in one launch.
//
// (a, b) -> factor * (a cos t - b sin t, b cos t + a sin t) for every pair of a head's first
// rotary_dim elements, t = 2 pi * position * f.  The frequency f comes as a 64-bit fixed-point
// fraction of a turn F = round(f * 2^64): position * F mod 2^64 is the fraction of a turn of
// the angle with an error of |position| / 2 * 2^-64 (the table is made in decimal arithmetic, so that F is
// the nearest number), where an fp32 angle would already be off by
// position * 2^-24 radians (0.06 at position 10^6).  The top 32 bits, read as a signed
// number, are the angle in half-open [-1/2, 1/2) turns; rounding them to fp32 costs 2^-24
// relative, like any fp32 cosine's own rounding.
//
// Bound: HBM (reads and writes each element once; 3 flops an element).  Angles are computed
// once per token and pair into shared memory and shared by all heads of the token; a thread
// then moves 16 bytes of each half of a pair at a time (8 bytes, or single elements, where
// sizes or strides leave no more).  Full occupancy hides the latency: 2 x 16001 tokens, 80 + 8
// heads of 128, bf16: 236 us (6.11 TB/s; in fp32 432 us, 6.67 TB/s, neighbouring pairs 446); 6 blocks an SM
// 264 us, 4 blocks 315; two rows in flight a thread (48 registers) 266, four 410.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "../../include/attn_bwd_b200.h"
#include "fast_div.h"
#include "host_shared.h"

namespace {

constexpr int kRopeThreads = 256, kRopeBlocks = 8;   // 8 blocks an SM: full of threads (32 registers each)
constexpr int kMaxTokens = 16;   // of a block

struct RopeParams {
  long long tokens;          // bs * seq
  int seq, q_heads, heads;   // heads = q_heads + k_heads
  int half;                  // rotary_dim / 2 pairs
  int pair_chunks, chunks;   // chunks of VEC pairs; with the chunks of the part that is copied
  int rotary_dim;
  int tok_per_block;
  attn_bwd::FastDiv div_heads, div_half, div_seq;
  float factor, sign;
  long long pos_stride;
  long long qi[3], ki[3], qo[3], ko[3];
  const long long* pos;
  const unsigned long long* turns;
  const void *q, *k;
  void *qo_p, *ko_p;
};

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f<float>(float x) { return x; }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }

template <typename T, int VEC>
struct Pack {
  alignas(VEC * sizeof(T)) T v[VEC];
};

// One block: tok_per_block tokens.  Thread (row, chunk): rows are (token, head) pairs.
// INTER: a chunk is VEC neighbouring elements (VEC / 2 pairs; VEC = 1 means one pair moved
// element by element).  Otherwise a chunk is VEC elements of the lower and VEC of the upper half.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kRopeThreads, kRopeBlocks) rope_kernel(const RopeParams p) {
  constexpr bool ONE = INTER && VEC > 1;        // a chunk is one piece of the row
  constexpr int PV = ONE ? VEC / 2 : VEC;       // pairs of a chunk
  extern __shared__ __align__(16) float2 cs[];  // [tok_per_block][half] cosine and sine, times the factor
  __shared__ long long offs[kMaxTokens][4];     // of a token in q, k, their results
  const long long tok0 = (long long)blockIdx.x * p.tok_per_block;
  const int ntok = int(min((long long)p.tok_per_block, p.tokens - tok0));
  const long long b0 = tok0 / p.seq;
  const int at0 = int(tok0 - b0 * p.seq);
  for (int i = threadIdx.x; i < ntok * p.half; i += kRopeThreads) {
    const int t = p.div_half.div(i), n = i - t * p.half;
    const int over = p.div_seq.div(at0 + t), at = at0 + t - over * p.seq;
    const long long b = b0 + over;
    const unsigned long long pos = (unsigned long long)p.pos[b * p.pos_stride + at];
    const int turn = int(unsigned((pos * p.turns[n] + 0x80000000ull) >> 32));
    float s, c;
    sincospif(float(turn) * 0x1p-31f, &s, &c);   // half turns
    // pairs 2m and 2m + 1 of all chunks lie together, so that neighbouring chunks' threads read
    // neighbouring 16 bytes
    const int c0 = n / PV, e = n - c0 * PV;
    cs[t * p.half + (PV > 1 ? ((e >> 1) * p.pair_chunks + c0) * 2 + (e & 1) : n)] =
        make_float2(c * p.factor, s * p.factor * p.sign);
    if (n == 0) {
      offs[t][0] = b * p.qi[0] + at * p.qi[2];
      offs[t][1] = b * p.ki[0] + at * p.ki[2];
      offs[t][2] = b * p.qo[0] + at * p.qo[2];
      offs[t][3] = b * p.ko[0] + at * p.ko[2];
    }
  }
  __syncthreads();
  const int rows = ntok * p.heads;
  const int per = kRopeThreads / p.chunks > 0 ? kRopeThreads / p.chunks : 1;   // rows at a time
  const int lanes = per * p.chunks;
  using V = Pack<T, VEC>;
  // more chunks than threads (heads of over 2000 elements): every thread takes several
  for (int c0 = threadIdx.x; c0 < (p.chunks > kRopeThreads ? p.chunks : lanes); c0 += kRopeThreads) {
    const int chunk = c0 % p.chunks;
    const bool copy = chunk >= p.pair_chunks;   // the part of the head that is not rotated
    const int lo = copy ? p.rotary_dim + (chunk - p.pair_chunks) * VEC
                        : INTER ? (VEC > 1 ? chunk * VEC : 2 * chunk) : chunk * VEC;
    const int hi = INTER ? 2 * chunk + 1 : p.half + chunk * VEC;
    for (int row = c0 / p.chunks; row < rows; row += per) {
      const int t = p.div_heads.div(row), h = row - t * p.heads;
      const bool isq = h < p.q_heads;
      const T* in = isq ? static_cast<const T*>(p.q) + offs[t][0] + h * p.qi[1]
                        : static_cast<const T*>(p.k) + offs[t][1] + (h - p.q_heads) * p.ki[1];
      T* out = isq ? static_cast<T*>(p.qo_p) + offs[t][2] + h * p.qo[1]
                   : static_cast<T*>(p.ko_p) + offs[t][3] + (h - p.q_heads) * p.ko[1];
      V x = *reinterpret_cast<const V*>(in + lo);
      if (!copy) {
        V y;
        if (!ONE) y = *reinterpret_cast<const V*>(in + hi);
        const float2* w = cs + t * p.half;
#pragma unroll
        for (int e = 0; e < PV; ++e) {
          float2 a;
          if (PV > 1) {
            const float4 f = *reinterpret_cast<const float4*>(w + ((e >> 1) * p.pair_chunks + chunk) * 2);
            a = (e & 1) ? make_float2(f.z, f.w) : make_float2(f.x, f.y);
          } else {
            a = w[chunk];
          }
          T& p0 = ONE ? x.v[(2 * e) % VEC] : x.v[e % VEC];
          T& p1 = ONE ? x.v[(2 * e + 1) % VEC] : y.v[e % VEC];
          const float u = to_f(p0), v = to_f(p1);
          p0 = from_f<T>(u * a.x - v * a.y);
          p1 = from_f<T>(v * a.x + u * a.y);
        }
        if (!ONE) *reinterpret_cast<V*>(out + hi) = y;
      }
      *reinterpret_cast<V*>(out + lo) = x;
    }
  }
}

template <typename T, int VEC>
cudaError_t launch_width(RopeParams p, int dim, bool inter, cudaStream_t stream) {
  p.pair_chunks = inter && VEC > 1 ? p.rotary_dim / VEC : p.half / VEC;
  p.chunks = p.pair_chunks + (dim - p.rotary_dim) / VEC;
  // A block's rows keep its threads busy for a few rounds; at most 16 KB of angles.  2 x 16001 tokens, 88
  // heads: 238 us; 248 with 96 rows a block, 247 with 720.  12 x 467 tokens: 53; 59 from 360 rows on.  (A few
  // tokens fill few blocks, whose threads take up to six rounds: 8 tokens of 88 heads are 4 blocks.)
  int tpb = 192 / p.heads;
  if (tpb > kMaxTokens) tpb = kMaxTokens;
  if ((long long)tpb * p.half * 8 > 16384) tpb = 16384 / (p.half * 8);
  if (tpb < 1) tpb = 1;
  p.tok_per_block = tpb;
  p.div_heads = attn_bwd::fast_div(p.heads);
  p.div_half = attn_bwd::fast_div(p.half);
  p.div_seq = attn_bwd::fast_div(p.seq);
  const long long blocks = (p.tokens + tpb - 1) / tpb;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  const size_t smem = size_t(tpb) * p.half * sizeof(float2);
  if (inter) rope_kernel<T, VEC, true><<<unsigned(blocks), kRopeThreads, smem, stream>>>(p);
  else rope_kernel<T, VEC, false><<<unsigned(blocks), kRopeThreads, smem, stream>>>(p);
  return cudaPeekAtLastError();
}

// align: bytes that every row's address is a multiple of (16, 8 or less).
// The widest pieces that fit: 2 x 16001 tokens take 238 us in pieces of 16 bytes, 308 of 8, 516 element by
// element; heads of 80 with 40 rotated take 59 us in pieces of 8 bytes, 130 element by element.
template <typename T>
cudaError_t launch_rope(const RopeParams& p, int dim, bool inter, int align, cudaStream_t stream) {
  constexpr int V16 = 16 / int(sizeof(T)), V8 = V16 / 2;
  const auto fits = [&](int v) { return p.rotary_dim % (inter ? v : 2 * v) == 0 && dim % v == 0; };
  if (align >= 16 && fits(V16)) return launch_width<T, V16>(p, dim, inter, stream);
  if (align >= 8 && fits(V8)) return launch_width<T, V8>(p, dim, inter, stream);
  return launch_width<T, 1>(p, dim, inter, stream);
}

// What every row's offset in bytes is a multiple of: 16, 8 or 1.
int stride_align(const int64_t* st, int bs, int heads, int seq, int es) {
  const int n[3] = {bs, heads, seq};
  int a = 16;
  for (int i = 0; i < 3; ++i)
    while (a > 1 && n[i] > 1 && (st[i] * es) % a) a = a == 16 ? 8 : 1;
  return a;
}
int pointer_align(const void* x, const void* y) {
  const uintptr_t u = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y);
  return (u & 15u) == 0 ? 16 : (u & 7u) == 0 ? 8 : 1;
}

}  // namespace

extern "C" int attn_bwd_b200_rope(const attn_bwd_rope_t* a, const void* q, const void* k, const int64_t* positions,
                                  const int64_t* turns, void* q_out, void* k_out, attn_bwd_stream_t stream) {
  if (!a || a->bs < 0 || a->seq < 0 || a->q_heads < 0 || a->k_heads < 0 || a->head_dim < 1 || a->rotary_dim < 2 ||
      a->rotary_dim > a->head_dim || a->rotary_dim % 2 || a->head_dim > 4096 || a->position_stride < 0 || a->seq > (1 << 30))
    return ATTN_BWD_EINVAL;
  if (a->dtype < ATTN_BWD_DT_BF16 || a->dtype > ATTN_BWD_DT_FP32) return ATTN_BWD_EUNSUPPORTED;
  if (a->q_heads > (1 << 20) || a->k_heads > (1 << 20)) return ATTN_BWD_EINVAL;
  if (a->bs == 0 || a->seq == 0 || a->q_heads + a->k_heads == 0) return ATTN_BWD_OK;
  if (!positions || !turns || (a->q_heads && (!q || !q_out)) || (a->k_heads && (!k || !k_out))) return ATTN_BWD_EINVAL;
  attn_bwd::HostDevice dev;
  const int rc = attn_bwd::host_device(&dev);
  if (rc) return rc;
  RopeParams p = {};
  p.tokens = (long long)a->bs * a->seq;
  p.seq = a->seq;
  p.q_heads = a->q_heads;
  p.heads = a->q_heads + a->k_heads;
  p.half = a->rotary_dim / 2;
  p.rotary_dim = a->rotary_dim;
  p.factor = a->factor;
  p.sign = a->inverse ? -1.f : 1.f;
  p.pos_stride = a->position_stride;
  const int es = a->dtype == ATTN_BWD_DT_FP32 ? 4 : 2;
  for (int i = 0; i < 3; ++i) {
    p.qi[i] = a->q_in[i];
    p.ki[i] = a->k_in[i];
    p.qo[i] = a->q_out[i];
    p.ko[i] = a->k_out[i];
  }
  int align = 16;
  const auto lower = [&](int x) { if (x < align) align = x; };
  if (a->q_heads) {
    lower(stride_align(a->q_in, a->bs, a->q_heads, a->seq, es));
    lower(stride_align(a->q_out, a->bs, a->q_heads, a->seq, es));
    lower(pointer_align(q, q_out));
  }
  if (a->k_heads) {
    lower(stride_align(a->k_in, a->bs, a->k_heads, a->seq, es));
    lower(stride_align(a->k_out, a->bs, a->k_heads, a->seq, es));
    lower(pointer_align(k, k_out));
  }
  p.pos = reinterpret_cast<const long long*>(positions);
  p.turns = reinterpret_cast<const unsigned long long*>(turns);
  p.q = q;
  p.k = k;
  p.qo_p = q_out;
  p.ko_p = k_out;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (a->dtype == ATTN_BWD_DT_BF16) e = launch_rope<__nv_bfloat16>(p, a->head_dim, a->interleaved != 0, align, s);
  else if (a->dtype == ATTN_BWD_DT_FP16) e = launch_rope<__half>(p, a->head_dim, a->interleaved != 0, align, s);
  else e = launch_rope<float>(p, a->head_dim, a->interleaved != 0, align, s);
  return e == cudaSuccess ? ATTN_BWD_OK : ATTN_BWD_ECUDA;
}
