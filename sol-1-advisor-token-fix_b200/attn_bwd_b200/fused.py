"""Attention with capped, biased and masked scores, forward and backward, without materialised
weights (``attn_bwd_b200_fused_fwd`` / ``_bwd``)."""
import ctypes
import math

import torch

from . import _lib

__all__ = ["fused_attn_fwd", "fused_attn_bwd"]

_TYPES = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_FP16}

_MIN_CAP = 1e-30   # the library's; checked before the number is narrowed to fp32, where far less is 0: no cap


def _check(t, name, like=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if t.device.type != "cuda":
        raise ValueError(f"{name}: tensor must be on a CUDA device (no CPU path), got {t.device}")
    if t.dim() != 4:
        raise ValueError(f"{name}: expected 4 dimensions, got {tuple(t.shape)}")
    if like is None:
        if t.dtype not in _TYPES:
            raise TypeError(f"{name}: expected bfloat16 or float16, got {t.dtype}")
    elif t.dtype != like.dtype:
        raise TypeError(f"{name}: expected dtype {like.dtype}, got {t.dtype}")
    elif t.device != like.device:
        raise ValueError(f"{name}: expected a tensor on {like.device}, got {t.device}")


def _ready(t):
    """The tensor, or a contiguous copy where its strides or its address do not fit the kernels'
    descriptors (head elements contiguous, other strides positive multiples of 8, 16-byte aligned)."""
    st, n = t.stride(), t.shape
    ok = st[3] == 1 and t.data_ptr() % 16 == 0 and all(
        n[i] <= 1 or (st[i] > 0 and st[i] % 8 == 0) for i in range(3))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _aux(t, name, dtype, shape, dev):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if t.device != dev:
        raise ValueError(f"{name}: expected a tensor on {dev}, got {t.device}")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected dtype {dtype}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    return t.contiguous()


def _bound(name, tensors, q, k, v, scale, softcap, slopes, causal, prefix_lens, documents):
    """The call through the C++ binding, or None where the general path has to look at it."""
    qd = kd = documents
    if isinstance(documents, (tuple, list)):
        if len(documents) != 2 or documents[0] is None or documents[1] is None:
            return None
        qd, kd = documents
    if scale is None:
        if not isinstance(q, torch.Tensor) or q.dim() != 4 or q.shape[3] == 0:
            return None
        scale = 1.0 / math.sqrt(q.shape[3])
    if not (0 < scale < math.inf and (softcap == 0 or _MIN_CAP < softcap < math.inf)):
        return None
    return _lib.bound(name, *tensors, scale, softcap, slopes, bool(causal), prefix_lens, qd, kd)


class _Call:
    """Checked arguments of one call: the C structure and the tensors that it points into."""

    def __init__(self, q, k, v, scale, softcap, slopes, causal, prefix_lens, documents):
        _check(q, "query_states")
        _check(k, "key_states", q)
        _check(v, "value_states", q)
        bs, h, sq, d = q.shape
        kvh, skv = k.shape[1], k.shape[2]
        if d not in (64, 128):
            raise ValueError(f"query_states: head_dim must be 64 or 128, got {d}")
        if tuple(k.shape) != (bs, kvh, skv, d) or tuple(v.shape) != tuple(k.shape):
            raise ValueError(f"key_states and value_states must be [{bs}, kv_heads, seq_kv, {d}], got "
                             f"{tuple(k.shape)} and {tuple(v.shape)}")
        if h < 1 or kvh < 1 or h % kvh:
            raise ValueError(f"{h} query heads cannot share {kvh} key heads")
        scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
        if not (scale > 0 and math.isfinite(scale)):
            raise ValueError(f"scale must be positive, got {scale}")
        softcap = float(softcap or 0.0)
        if not (softcap == 0 or _MIN_CAP < softcap < math.inf):
            raise ValueError(f"softcap must be above {_MIN_CAP} and finite, or 0 for none, got {softcap}")
        if prefix_lens is not None and not causal:
            raise ValueError("prefix_lens needs causal=True: without it every query sees all keys")
        dev = q.device
        self.device = dev
        self.q, self.k, self.v = _ready(q), _ready(k), _ready(v)
        self.keep = []
        a = self.args = _lib.FusedArgs()
        a.bs, a.seq_q, a.seq_kv, a.heads, a.kv_heads, a.head_dim = bs, sq, skv, h, kvh, d
        a.dtype, a.causal, a.scale, a.softcap = _TYPES[q.dtype], int(bool(causal)), scale, softcap
        if slopes is not None:
            a.slopes = self._hold(_aux(slopes, "slopes", torch.float32, (h,), dev))
        if prefix_lens is not None:
            a.prefix_lens = self._hold(_aux(prefix_lens, "prefix_lens", torch.int32, (bs,), dev))
        if documents is not None:
            if isinstance(documents, torch.Tensor):
                if sq != skv:
                    raise ValueError("documents: give a pair (of queries, of keys) where their numbers differ")
                documents = (documents, documents)
            if not isinstance(documents, (tuple, list)) or len(documents) != 2:
                raise ValueError("documents: expected a tensor or a pair (of queries, of keys)")
            a.q_documents = self._hold(_aux(documents[0], "documents of queries", torch.int32, (bs, sq), dev))
            a.kv_documents = self._hold(_aux(documents[1], "documents of keys", torch.int32, (bs, skv), dev))
        for t, dst in zip((self.q, self.k, self.v), (a.q_stride, a.k_stride, a.v_stride)):
            dst[:] = t.stride()[:3]

    def _hold(self, t):
        self.keep.append(t)
        return t.data_ptr()

    def workspace(self, backward):
        n = _lib.load().attn_bwd_b200_fused_workspace(ctypes.byref(self.args), backward)
        if n < 0:
            raise _lib.AttnBwdError("attn_bwd_b200_fused_workspace", -n)
        return (torch.empty(n, dtype=torch.uint8, device=self.device) if n else None), n


def fused_attn_fwd(query_states, key_states, value_states, scale=None, softcap=0.0, slopes=None, causal=False,
                   prefix_lens=None, documents=None):
    """Attention forward.  Returns (attn_output [bs, seq_q, heads, d], lse [bs, heads, seq_q] float32).

    query_states [bs, heads, seq_q, d], key_states and value_states [bs, kv_heads, seq_kv, d], bfloat16 or
    float16, d 64 or 128, heads a multiple of kv_heads, batch and heads at most 65535; any strides
    (copied only where head elements are not contiguous or rows not 16-byte aligned).  The queries are
    the last seq_q positions: one row of queries over a long cache is a decoding step.

    The score of head h, query position i and key j is x = scale * q.k (default scale
    1 / sqrt(d)), capped to softcap * tanh(x / softcap) if softcap is not 0 (then above 1e-30), minus
    slopes[h] * |i - j| (slopes [heads] float32: constants, no gradient is taken).  A query sees
      - with ``causal``, keys j <= i, and all keys j < prefix_lens[b] (int32 [bs]) besides;
      - with ``documents`` (int32 [bs, seq], or a pair for queries and keys), keys of its own
        document.  Negative numbers are padding: such queries and keys belong to no document, and
        what they hold (NaN included) reaches no result.
    A query that sees no key has output 0 and lse -inf.  A NaN or infinity in a query, key or value of
    a document (or without documents) may reach all results near it, seen or not.

    Weights are rounded to the inputs' 16 bits before they are multiplied with the values; scores, their
    maxima and sums, lse and the products' sums are float32.  There is no dropout: a layer that drops weights
    keeps them, and :func:`attn_bwd` takes its gradients."""
    softcap = softcap or 0.0
    mods = (query_states, key_states, value_states, scale, softcap, slopes, causal, prefix_lens, documents)
    r = _bound("fused_fwd", (query_states, key_states, value_states), *mods)
    if r is not None:
        return r
    c = _Call(*mods)
    bs, h, sq, d = query_states.shape
    with torch.cuda.device(c.device):
        o = torch.empty((bs, sq, h, d), dtype=query_states.dtype, device=c.device)
        lse = torch.empty((bs, h, sq), dtype=torch.float32, device=c.device)
        ws, n = c.workspace(0)
        _lib.call("attn_bwd_b200_fused_fwd", ctypes.byref(c.args), c.q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(),
                  o.data_ptr(), lse.data_ptr(), ws.data_ptr() if n else 0, n, torch.cuda.current_stream().cuda_stream)
    return o, lse


def fused_attn_bwd(grad_attn_output, query_states, key_states, value_states, attn_output, lse, scale=None, softcap=0.0,
                   slopes=None, causal=False, prefix_lens=None, documents=None):
    """Gradients (grad_query, grad_key, grad_value) of :func:`fused_attn_fwd`'s first three
    arguments, from grad_attn_output [bs, seq_q, heads, d] and that call's results; the other
    arguments as they were given there.  The gradients have the shapes of the states (keys' and
    values' summed over the heads that share them) and their order in memory.  At most
    33554432 keys; with documents, at most 262144 positions.  Equal inputs give equal bits.

    attn_output and lse have to be that very call's: queries whose keys all lie in one tile of 128 do not
    read attn_output, so results merged from calls over parts of the keys give wrong gradients.  The
    weights and the gradients of the scores are rounded to 16 bits before they are multiplied.  In float16 a
    gradient of a score below 6e-8 is lost and one above 65504 infinite, also where the results would
    be in range: scale the loss, as for any float16 gradient."""
    softcap = softcap or 0.0
    mods = (query_states, key_states, value_states, scale, softcap, slopes, causal, prefix_lens, documents)
    r = _bound("fused_bwd", (grad_attn_output, query_states, key_states, value_states, attn_output, lse), *mods)
    if r is not None:
        return r
    c = _Call(*mods)
    bs, h, sq, d = query_states.shape
    _check(grad_attn_output, "grad_attn_output", query_states)
    _check(attn_output, "attn_output", query_states)
    for t, name in ((grad_attn_output, "grad_attn_output"), (attn_output, "attn_output")):
        if tuple(t.shape) != (bs, sq, h, d):
            raise ValueError(f"{name}: expected shape {(bs, sq, h, d)}, got {tuple(t.shape)}")
    with torch.cuda.device(c.device):
        lse = _aux(lse, "lse", torch.float32, (bs, h, sq), c.device)
        do, o = (t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
                 for t in (grad_attn_output, attn_output))
        grads = []
        for t, dst in ((c.q, c.args.dq_stride), (c.k, c.args.dk_stride), (c.v, c.args.dv_stride)):
            g = torch.empty_like(t)
            if g.stride(3) != 1:
                g = torch.empty(t.shape, dtype=t.dtype, device=t.device)
            dst[:] = g.stride()[:3]
            grads.append(g)
        dq, dk, dv = grads
        ws, n = c.workspace(1)
        _lib.call("attn_bwd_b200_fused_bwd", ctypes.byref(c.args), do.data_ptr(), c.q.data_ptr(), c.k.data_ptr(),
                  c.v.data_ptr(), o.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                  ws.data_ptr() if n else 0, n, torch.cuda.current_stream().cuda_stream)
    return dq, dk, dv
