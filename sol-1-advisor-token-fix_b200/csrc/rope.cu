// rope.cu — rotary positions of queries and keys (and of their gradients) in one launch.
//
// (a, b) -> factor * (a cos t - b sin t, b cos t + a sin t) for every pair of a head's first
// rotary_dim elements, t = 2 pi * position * f.  The frequency f comes as a 64-bit fixed-point
// fraction of a turn F = round(f * 2^64): position * F mod 2^64 is the fraction of a turn of
// the angle with an error of position / 2 * 2^-64, where an fp32 angle would already be off by
// position * 2^-24 radians (0.06 at position 10^6).  The top 32 bits, read as a signed
// number, are the angle in half-open [-1/2, 1/2) turns; rounding them to fp32 costs 2^-24
// relative, like any fp32 cosine's own rounding.
//
// Bound: HBM (reads and writes each element once; 3 flops an element).  Angles are computed
// once per token and pair into shared memory and shared by all heads of the token; a thread
// then moves 16 bytes of each half of a pair at a time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "../../include/attn_bwd_b200.h"
#include "host_shared.h"

namespace {

constexpr int kRopeThreads = 256;

struct RopeParams {
  long long tokens;          // bs * seq
  int seq, q_heads, heads;   // heads = q_heads + k_heads
  int half;                  // rotary_dim / 2 pairs
  int pair_chunks, chunks;   // chunks of VEC pairs; with the chunks of the part that is copied
  int rotary_dim;
  int tok_per_block;
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
  static_assert(VEC == 1 || VEC * sizeof(T) == 16, "one element or 16 bytes");
  alignas(VEC == 1 ? alignof(T) : 16) T v[VEC];
};

// One block: tok_per_block tokens.  Thread (row, chunk): rows are (token, head) pairs.
// INTER: a chunk is VEC neighbouring elements (VEC / 2 pairs; VEC = 1 means one pair moved
// element by element).  Otherwise a chunk is VEC elements of the lower and VEC of the upper half.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeParams p) {
  extern __shared__ float2 cs[];   // [tok_per_block][half] cosine and sine, times the factor
  const long long tok0 = (long long)blockIdx.x * p.tok_per_block;
  const int ntok = int(min((long long)p.tok_per_block, p.tokens - tok0));
  for (int i = threadIdx.x; i < ntok * p.half; i += kRopeThreads) {
    const int t = i / p.half, n = i - t * p.half;
    const long long tok = tok0 + t, b = tok / p.seq;
    const unsigned long long pos = (unsigned long long)p.pos[b * p.pos_stride + (tok - b * p.seq)];
    const int turn = int(unsigned((pos * p.turns[n] + 0x80000000ull) >> 32));
    float s, c;
    sincospif(float(turn) * 0x1p-31f, &s, &c);   // half turns
    cs[i] = make_float2(c * p.factor, s * p.factor * p.sign);
  }
  __syncthreads();
  const int rows = ntok * p.heads;
  const int per = kRopeThreads / p.chunks > 0 ? kRopeThreads / p.chunks : 1;   // rows at a time
  const int lanes = per * p.chunks;
  // more chunks than threads (heads of over 2000 elements): every thread takes several
  for (int c0 = threadIdx.x; c0 < (p.chunks > kRopeThreads ? p.chunks : lanes); c0 += kRopeThreads) {
    const int chunk = c0 % p.chunks;
#pragma unroll 4
    for (int row = c0 / p.chunks; row < rows; row += per) {
      const int t = row / p.heads, h = row - t * p.heads;
      const long long tok = tok0 + t, b = tok / p.seq, s = tok - b * p.seq;
      const bool isq = h < p.q_heads;
      const int hh = isq ? h : h - p.q_heads;
      const T* in = isq ? static_cast<const T*>(p.q) + b * p.qi[0] + hh * p.qi[1] + s * p.qi[2]
                        : static_cast<const T*>(p.k) + b * p.ki[0] + hh * p.ki[1] + s * p.ki[2];
      T* out = isq ? static_cast<T*>(p.qo_p) + b * p.qo[0] + hh * p.qo[1] + s * p.qo[2]
                   : static_cast<T*>(p.ko_p) + b * p.ko[0] + hh * p.ko[1] + s * p.ko[2];
      using V = Pack<T, VEC>;
      if (chunk >= p.pair_chunks) {   // the part of the head that is not rotated
        const int e = p.rotary_dim + (chunk - p.pair_chunks) * VEC;
        *reinterpret_cast<V*>(out + e) = *reinterpret_cast<const V*>(in + e);
        continue;
      }
      const float2* w = cs + t * p.half;
      if (INTER && VEC > 1) {
        const int e = chunk * VEC;
        V x = *reinterpret_cast<const V*>(in + e);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
          const float2 a = w[e / 2 + i];
          const float u = to_f(x.v[2 * i]), v = to_f(x.v[(2 * i + 1) % VEC]);
          x.v[2 * i] = from_f<T>(u * a.x - v * a.y);
          x.v[(2 * i + 1) % VEC] = from_f<T>(v * a.x + u * a.y);
        }
        *reinterpret_cast<V*>(out + e) = x;
      } else {
        const int lo = INTER ? 2 * chunk : chunk * VEC, hi = INTER ? 2 * chunk + 1 : p.half + chunk * VEC;
        V x = *reinterpret_cast<const V*>(in + lo), y = *reinterpret_cast<const V*>(in + hi);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float2 a = w[chunk * VEC + i];
          const float u = to_f(x.v[i]), v = to_f(y.v[i]);
          x.v[i] = from_f<T>(u * a.x - v * a.y);
          y.v[i] = from_f<T>(v * a.x + u * a.y);
        }
        *reinterpret_cast<V*>(out + lo) = x;
        *reinterpret_cast<V*>(out + hi) = y;
      }
    }
  }
}

template <typename T>
cudaError_t launch_rope(RopeParams p, int dim, bool inter, bool vec_ok, cudaStream_t stream) {
  constexpr int VEC = 16 / int(sizeof(T));
  const bool vec = vec_ok && p.rotary_dim % (inter ? VEC : 2 * VEC) == 0 && dim % VEC == 0;
  const int ve = vec ? VEC : 1;
  p.pair_chunks = inter && vec ? p.rotary_dim / VEC : p.half / ve;
  p.chunks = p.pair_chunks + (dim - p.rotary_dim) / ve;
  // a block's rows keep its threads busy for a few rounds; at most 16 KB of angles
  int tpb = 192 / p.heads;
  if (tpb > 16) tpb = 16;
  if ((long long)tpb * p.half * 8 > 16384) tpb = 16384 / (p.half * 8);
  if (tpb < 1) tpb = 1;
  p.tok_per_block = tpb;
  const long long blocks = (p.tokens + tpb - 1) / tpb;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  const size_t smem = size_t(tpb) * p.half * sizeof(float2);
  if (vec)
    inter ? rope_kernel<T, VEC, true><<<unsigned(blocks), kRopeThreads, smem, stream>>>(p)
          : rope_kernel<T, VEC, false><<<unsigned(blocks), kRopeThreads, smem, stream>>>(p);
  else
    inter ? rope_kernel<T, 1, true><<<unsigned(blocks), kRopeThreads, smem, stream>>>(p)
          : rope_kernel<T, 1, false><<<unsigned(blocks), kRopeThreads, smem, stream>>>(p);
  return cudaPeekAtLastError();
}

// Element offsets of every row: 16-byte multiples, so that a row can be moved in 16-byte words.
bool strides_ok16(const int64_t* st, int bs, int heads, int seq, int es) {
  const int n[3] = {bs, heads, seq};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (st[i] * es) % 16) return false;
  return true;
}

}  // namespace

extern "C" int attn_bwd_b200_rope(const attn_bwd_rope_t* a, const void* q, const void* k, const int64_t* positions,
                                  const int64_t* turns, void* q_out, void* k_out, attn_bwd_stream_t stream) {
  if (!a || a->bs < 0 || a->seq < 0 || a->q_heads < 0 || a->k_heads < 0 || a->head_dim < 1 || a->rotary_dim < 2 ||
      a->rotary_dim > a->head_dim || a->rotary_dim % 2 || a->head_dim > 4096 || a->position_stride < 0)
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
  bool vec = true;
  for (int i = 0; i < 3; ++i) {
    p.qi[i] = a->q_in[i];
    p.ki[i] = a->k_in[i];
    p.qo[i] = a->q_out[i];
    p.ko[i] = a->k_out[i];
  }
  if (a->q_heads)
    vec = vec && strides_ok16(a->q_in, a->bs, a->q_heads, a->seq, es) &&
          strides_ok16(a->q_out, a->bs, a->q_heads, a->seq, es) &&
          ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out)) & 15u) == 0;
  if (a->k_heads)
    vec = vec && strides_ok16(a->k_in, a->bs, a->k_heads, a->seq, es) &&
          strides_ok16(a->k_out, a->bs, a->k_heads, a->seq, es) &&
          ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_out)) & 15u) == 0;
  p.pos = reinterpret_cast<const long long*>(positions);
  p.turns = reinterpret_cast<const unsigned long long*>(turns);
  p.q = q;
  p.k = k;
  p.qo_p = q_out;
  p.ko_p = k_out;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (a->dtype == ATTN_BWD_DT_BF16) e = launch_rope<__nv_bfloat16>(p, a->head_dim, a->interleaved != 0, vec, s);
  else if (a->dtype == ATTN_BWD_DT_FP16) e = launch_rope<__half>(p, a->head_dim, a->interleaved != 0, vec, s);
  else e = launch_rope<float>(p, a->head_dim, a->interleaved != 0, vec, s);
  return e == cudaSuccess ? ATTN_BWD_OK : ATTN_BWD_ECUDA;
}
