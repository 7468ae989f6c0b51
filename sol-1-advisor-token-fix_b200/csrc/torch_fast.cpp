// torch_fast.cpp — host binding for PyTorch callers of the full call.
//
// The same work as the Python fast path of attn_bwd_b200.attn_bwd (input checks,
// output allocation, the caller's current stream, the C-ABI call), done in C++ so a
// call costs a few microseconds of host time instead of ~12.  It calls the C-ABI
// entry point attn_bwd_b200 (include/attn_bwd_b200.h) and nothing else; the kernels
// live in libattn_bwd_b200.so.
//
// fast(dO, P, Pd, V, M, p) returns
//   (dS, dV)  on success,
//   an int    (the library's error code) when the call was made and failed,
//   None      when the inputs need the general path (other dtypes / shapes / strides /
//             devices, misaligned pointers): the Python side then converts and calls
//             the library through ctypes.
// rope, fused_fwd and fused_bwd do the same for the rotary positions and the fused attention:
// a decoding step's calls are shorter than the Python path's checks (30 us of it a call).
#include <algorithm>

#include <torch/extension.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>

#include "../../include/attn_bwd_b200.h"

namespace {

constexpr int64_t kHeads = 80, kKvHeads = 8, kHeadDim = 128;

inline bool dense16(const at::Tensor& t) {
  return t.is_contiguous() && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
}

py::object fast(const at::Tensor& dO, const at::Tensor& P, const at::Tensor& Pd, const at::Tensor& V,
                const at::Tensor& M, double p) {
  if (!dO.is_cuda() || dO.scalar_type() != at::kBFloat16 || P.scalar_type() != at::kBFloat16 ||
      Pd.scalar_type() != at::kBFloat16 || V.scalar_type() != at::kBFloat16 || M.scalar_type() != at::kBool)
    return py::none();
  if (dO.dim() != 4 || V.dim() != 4 || P.dim() != 4 || Pd.dim() != 4 || M.dim() != 4) return py::none();
  const int64_t bs = dO.size(0), sq = dO.size(1), skv = V.size(2);
  if (dO.size(2) != kHeads || dO.size(3) != kHeadDim) return py::none();
  if (V.size(0) != bs || V.size(1) != kKvHeads || V.size(3) != kHeadDim) return py::none();
  const at::IntArrayRef ps = P.sizes();
  if (ps[0] != bs || ps[1] != kHeads || ps[2] != sq || ps[3] != skv || Pd.sizes() != ps || M.sizes() != ps)
    return py::none();
  const c10::Device dev = dO.device();
  if (P.device() != dev || Pd.device() != dev || V.device() != dev || M.device() != dev) return py::none();
  if (!dense16(dO) || !dense16(P) || !dense16(Pd) || !dense16(V) || !dense16(M)) return py::none();
  if (bs > INT32_MAX || sq > INT32_MAX || skv > INT32_MAX) return py::none();

  c10::cuda::OptionalCUDAGuard guard;
  if (dev.index() != c10::cuda::current_device()) guard.set_device(dev);
  at::Tensor dS = at::empty_like(P);
  at::Tensor dV = at::empty_like(V);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  const int rc = attn_bwd_b200(dO.data_ptr(), P.data_ptr(), Pd.data_ptr(), V.data_ptr(),
                               static_cast<const uint8_t*>(M.data_ptr()), static_cast<float>(p), int(bs), int(sq),
                               int(skv), dS.data_ptr(), dV.data_ptr(), reinterpret_cast<attn_bwd_stream_t>(stream));
  if (rc != 0) return py::int_(rc);
  return py::make_tuple(dS, dV);
}


// Sets the tensor's device for the scope if it is not the current one.
struct DeviceScope {
  c10::cuda::OptionalCUDAGuard guard;
  explicit DeviceScope(c10::Device dev) {
    if (dev.index() != c10::cuda::current_device()) guard.set_device(dev);
  }
};

inline attn_bwd_stream_t stream_of(c10::Device dev) {
  return reinterpret_cast<attn_bwd_stream_t>(c10::cuda::getCurrentCUDAStream(dev.index()).stream());
}

inline void set_strides(int64_t* dst, const at::Tensor& t) {
  for (int i = 0; i < 3; ++i) dst[i] = t.stride(i);
}

inline bool int_sizes(const at::Tensor& t) {
  for (int64_t n : t.sizes())
    if (n > INT32_MAX) return false;
  return true;
}

using OptTensor = std::optional<at::Tensor>;

// Whether results that the caller gave may be written: see _overlap and _check_places in rope.py, whose
// answer this repeats where it is yes (otherwise the general path says what is wrong).
struct Term {
  int64_t stride, lo, hi;
};
// Whether target is a sum of t * stride, lo <= t <= hi, strides falling; budget: see _reaches.
bool reaches(const Term* t, int n, int64_t target, int& budget) {
  if (n == 0) return target == 0;
  int64_t lo = 0, hi = 0;
  for (int i = 1; i < n; ++i) { lo += t[i].stride * t[i].lo; hi += t[i].stride * t[i].hi; }
  const auto floor_div = [](int64_t a, int64_t b) { return a >= 0 ? a / b : -((b - 1 - a) / b); };
  const int64_t last = std::min(t->hi, floor_div(target - lo, t->stride));
  for (int64_t k = std::max(t->lo, -floor_div(hi - target, t->stride)); k <= last; ++k)
    if (--budget < 0 || reaches(t + 1, n - 1, target - k * t->stride, budget)) return true;
  return false;
}
int64_t extent(const at::Tensor& t) {
  int64_t n = 1;
  for (int i = 0; i < 4; ++i) n += (t.size(i) - 1) * t.stride(i);
  return n;
}
bool overlap(const at::Tensor& x, const at::Tensor& y) {
  if (x.numel() == 0 || y.numel() == 0) return false;
  const int64_t es = x.element_size();
  const int64_t at = static_cast<char*>(y.data_ptr()) - static_cast<char*>(x.data_ptr());
  if (at >= extent(x) * es || -at >= extent(y) * es) return false;
  if (at % es) return true;
  Term t[8];
  int n = 0;
  for (int side = 0; side < 2; ++side)
    for (int i = 0; i < 4; ++i) {
      const at::Tensor& z = side ? y : x;
      const int64_t len = z.size(i) - 1, st = z.stride(i);
      if (len == 0 || st == 0) continue;
      int k = 0;
      while (k < n && t[k].stride != st) ++k;
      if (k == n) t[n++] = {st, 0, 0};
      (side ? t[k].lo : t[k].hi) += side ? -len : len;
    }
  std::sort(t, t + n, [](const Term& a, const Term& b) { return a.stride > b.stride; });
  int budget = 4096;
  return reaches(t, n, at / es, budget);
}
// Every step passes what the smaller ones reach.
bool nested(const at::Tensor& t) {
  int order[4] = {0, 1, 2, 3};
  std::sort(order, order + 4, [&](int a, int b) { return t.stride(a) < t.stride(b); });
  int64_t reach = 0;
  for (int i : order) {
    if (t.size(i) <= 1) continue;
    if (t.stride(i) <= reach) return false;
    reach += (t.size(i) - 1) * t.stride(i);
  }
  return true;
}
bool same_place(const at::Tensor& x, const at::Tensor& y) {
  if (x.data_ptr() != y.data_ptr()) return false;
  for (int i = 0; i < 4; ++i)
    if (x.size(i) > 1 && x.stride(i) != y.stride(i)) return false;
  return true;
}
bool places_ok(const at::Tensor& q, const at::Tensor& k, const OptTensor& qo, const OptTensor& ko) {
  const at::Tensor* in[2] = {&q, &k};
  const OptTensor* out[2] = {&qo, &ko};
  bool own[2];
  for (int i = 0; i < 2; ++i) {
    const OptTensor& o = *out[i];
    if (o.has_value() && (o->sizes() != in[i]->sizes() || o->scalar_type() != in[i]->scalar_type() ||
                          o->device() != in[i]->device() || o->stride(3) != 1 || !nested(*o)))
      return false;
    own[i] = o.has_value() && same_place(*o, *in[i]);
  }
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2; ++j)
      if (out[i]->has_value() && !own[j] && overlap(**out[i], *in[j])) return false;
  return !(qo.has_value() && ko.has_value() && overlap(*qo, *ko));
}

// rope(q, k, positions, turns, rotary_dim, factor, interleaved, inverse) and rope_into(.., q_out, k_out):
// two tensors of one type, int64 positions and turns that are contiguous; results in new tensors where
// none are given.
py::object rope_into(const at::Tensor& q, const at::Tensor& k, const at::Tensor& pos, const at::Tensor& turns,
                     int64_t rotary_dim, double factor, bool interleaved, bool inverse, const OptTensor& q_out,
                     const OptTensor& k_out) {
  if (!q.is_cuda() || q.dim() != 4 || k.dim() != 4 || q.scalar_type() != k.scalar_type()) return py::none();
  int dtype;
  switch (q.scalar_type()) {
    case at::kBFloat16: dtype = ATTN_BWD_DT_BF16; break;
    case at::kHalf: dtype = ATTN_BWD_DT_FP16; break;
    case at::kFloat: dtype = ATTN_BWD_DT_FP32; break;
    default: return py::none();
  }
  const int64_t bs = q.size(0), seq = q.size(2), d = q.size(3);
  if (k.size(0) != bs || k.size(2) != seq || k.size(3) != d || rotary_dim > d || !int_sizes(q) || !int_sizes(k))
    return py::none();
  const c10::Device dev = q.device();
  if (k.device() != dev || pos.device() != dev || turns.device() != dev) return py::none();
  if (q.stride(3) != 1 || k.stride(3) != 1) return py::none();
  if (pos.scalar_type() != at::kLong || !pos.is_contiguous()) return py::none();
  if (turns.scalar_type() != at::kLong || turns.dim() != 1 || turns.size(0) * 2 != rotary_dim || !turns.is_contiguous())
    return py::none();
  int64_t pstride = 0;
  if (pos.dim() == 2 && pos.size(1) == seq && (pos.size(0) == bs || pos.size(0) == 1)) pstride = pos.size(0) == 1 ? 0 : seq;
  else if (pos.dim() != 1 || pos.size(0) != seq) return py::none();
  DeviceScope scope(dev);
  if ((q_out.has_value() || k_out.has_value()) && !places_ok(q, k, q_out, k_out)) return py::none();
  at::Tensor qo = q_out.has_value() ? *q_out : at::empty_like(q), ko = k_out.has_value() ? *k_out : at::empty_like(k);
  if (qo.stride(3) != 1 || ko.stride(3) != 1) return py::none();
  attn_bwd_rope_t a = {};
  a.bs = int(bs);
  a.seq = int(seq);
  a.q_heads = int(q.size(1));
  a.k_heads = int(k.size(1));
  a.head_dim = int(d);
  a.rotary_dim = int(rotary_dim);
  a.dtype = dtype;
  a.interleaved = interleaved;
  a.inverse = inverse;
  a.factor = float(factor);
  a.position_stride = pstride;
  set_strides(a.q_in, q);
  set_strides(a.k_in, k);
  set_strides(a.q_out, qo);
  set_strides(a.k_out, ko);
  const int rc = attn_bwd_b200_rope(&a, q.data_ptr(), k.data_ptr(), pos.data_ptr<int64_t>(), turns.data_ptr<int64_t>(),
                                    qo.data_ptr(), ko.data_ptr(), stream_of(dev));
  if (rc != 0) return py::int_(rc);
  return py::make_tuple(qo, ko);
}

py::object rope(const at::Tensor& q, const at::Tensor& k, const at::Tensor& pos, const at::Tensor& turns,
                int64_t rotary_dim, double factor, bool interleaved, bool inverse) {
  return rope_into(q, k, pos, turns, rotary_dim, factor, interleaved, inverse, std::nullopt, std::nullopt);
}

// A state that the kernels read in place: see _ready in fused.py.
inline bool ready_state(const at::Tensor& t, const at::Tensor& q) {
  if (!t.is_cuda() || t.dim() != 4 || t.scalar_type() != q.scalar_type() || t.device() != q.device()) return false;
  if (t.stride(3) != 1 || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) || !int_sizes(t)) return false;
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1 && (t.stride(i) <= 0 || t.stride(i) % 8)) return false;
  return true;
}

inline bool aux(const OptTensor& t, at::ScalarType type, at::IntArrayRef shape, c10::Device dev, const void** out) {
  if (!t.has_value()) return true;
  if (t->device() != dev || t->scalar_type() != type || t->sizes() != shape || !t->is_contiguous()) return false;
  *out = t->data_ptr();
  return true;
}

// Fills the arguments; false where the general path has to look at them.
bool fused_args(attn_bwd_fused_t& a, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, double scale,
                double softcap, const OptTensor& slopes, bool causal, const OptTensor& prefix, const OptTensor& qdoc,
                const OptTensor& kdoc) {
  if (!ready_state(q, q) || !ready_state(k, q) || !ready_state(v, q)) return false;
  if (q.scalar_type() == at::kBFloat16) a.dtype = ATTN_BWD_DT_BF16;
  else if (q.scalar_type() == at::kHalf) a.dtype = ATTN_BWD_DT_FP16;
  else return false;
  const int64_t bs = q.size(0), h = q.size(1), sq = q.size(2), d = q.size(3), kv = k.size(1), skv = k.size(2);
  if (k.size(0) != bs || k.size(3) != d || v.sizes() != k.sizes() || (d != 64 && d != 128) || kv < 1 || h < 1 || h % kv)
    return false;
  const c10::Device dev = q.device();
  const void *sl = nullptr, *pr = nullptr, *qd = nullptr, *kd = nullptr;
  if (!aux(slopes, at::kFloat, {h}, dev, &sl) || !aux(prefix, at::kInt, {bs}, dev, &pr) ||
      !aux(qdoc, at::kInt, {bs, sq}, dev, &qd) || !aux(kdoc, at::kInt, {bs, skv}, dev, &kd) ||
      qdoc.has_value() != kdoc.has_value() || (prefix.has_value() && !causal))
    return false;
  a.bs = int(bs);
  a.seq_q = int(sq);
  a.seq_kv = int(skv);
  a.heads = int(h);
  a.kv_heads = int(kv);
  a.head_dim = int(d);
  a.causal = causal;
  a.scale = float(scale);
  a.softcap = float(softcap);
  a.slopes = static_cast<const float*>(sl);
  a.prefix_lens = static_cast<const int32_t*>(pr);
  a.q_documents = static_cast<const int32_t*>(qd);
  a.kv_documents = static_cast<const int32_t*>(kd);
  set_strides(a.q_stride, q);
  set_strides(a.k_stride, k);
  set_strides(a.v_stride, v);
  return true;
}

py::object fused_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, double scale, double softcap,
                     const OptTensor& slopes, bool causal, const OptTensor& prefix, const OptTensor& qdoc,
                     const OptTensor& kdoc) {
  attn_bwd_fused_t a = {};
  if (!fused_args(a, q, k, v, scale, softcap, slopes, causal, prefix, qdoc, kdoc)) return py::none();
  const c10::Device dev = q.device();
  DeviceScope scope(dev);
  at::Tensor o = at::empty({a.bs, a.seq_q, a.heads, a.head_dim}, q.options());
  at::Tensor lse = at::empty({a.bs, a.heads, a.seq_q}, q.options().dtype(at::kFloat));
  const int64_t n = attn_bwd_b200_fused_workspace(&a, 0);
  if (n < 0) return py::int_(-n);
  at::Tensor ws;
  if (n) ws = at::empty({n}, q.options().dtype(at::kByte));
  const int rc = attn_bwd_b200_fused_fwd(&a, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr<float>(),
                                         n ? ws.data_ptr() : nullptr, n, stream_of(dev));
  if (rc != 0) return py::int_(rc);
  return py::make_tuple(o, lse);
}

py::object fused_bwd(const at::Tensor& go, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                     const at::Tensor& o, const at::Tensor& lse, double scale, double softcap, const OptTensor& slopes,
                     bool causal, const OptTensor& prefix, const OptTensor& qdoc, const OptTensor& kdoc) {
  attn_bwd_fused_t a = {};
  if (!fused_args(a, q, k, v, scale, softcap, slopes, causal, prefix, qdoc, kdoc)) return py::none();
  const int64_t bs = a.bs, sq = a.seq_q, h = a.heads, d = a.head_dim;
  const c10::Device dev = q.device();
  for (const at::Tensor* t : {&go, &o})
    if (t->device() != dev || t->scalar_type() != q.scalar_type() || t->sizes() != at::IntArrayRef({bs, sq, h, d}) ||
        !dense16(*t))
      return py::none();
  if (lse.device() != dev || lse.scalar_type() != at::kFloat || lse.sizes() != at::IntArrayRef({bs, h, sq}) ||
      !lse.is_contiguous())
    return py::none();
  DeviceScope scope(dev);
  at::Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
  if (!ready_state(dq, q) || !ready_state(dk, q) || !ready_state(dv, q)) return py::none();
  set_strides(a.dq_stride, dq);
  set_strides(a.dk_stride, dk);
  set_strides(a.dv_stride, dv);
  const int64_t n = attn_bwd_b200_fused_workspace(&a, 1);
  if (n < 0) return py::int_(-n);
  at::Tensor ws;
  if (n) ws = at::empty({n}, q.options().dtype(at::kByte));
  const int rc = attn_bwd_b200_fused_bwd(&a, go.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                         lse.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                         n ? ws.data_ptr() : nullptr, n, stream_of(dev));
  if (rc != 0) return py::int_(rc);
  return py::make_tuple(dq, dk, dv);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "C++ host binding of the attn_bwd_b200 full call for PyTorch tensors";
  m.def("fast", &fast, "full call on ready inputs: (dS, dV), an error code, or None");
  m.def("rope", &rope, "rotary positions of ready inputs: (q, k), an error code, or None");
  m.def("rope_into", &rope_into, "the same into given results (either may be None)");
  m.def("fused_fwd", &fused_fwd, "fused attention on ready inputs: (o, lse), an error code, or None");
  m.def("fused_bwd", &fused_bwd, "its gradients: (dq, dk, dv), an error code, or None");
}
