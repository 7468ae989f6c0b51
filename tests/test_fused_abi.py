"""The C entry points of the fused attention with layouts that the Python calls never choose."""
import ctypes

import pytest
import torch

import attn_bwd_b200 as ab
from attn_bwd_b200 import _lib
from test_fused import _inputs

BF, HF = torch.bfloat16, torch.float16


def _place(shape, strides, offset, dtype):
    """A tensor of that shape and those strides (in elements) in a buffer of sevens, from an element on."""
    n = offset + sum((s - 1) * st for s, st in zip(shape, strides)) + 64
    buf = torch.full((n,), 7.0, dtype=dtype, device="cuda")
    assert buf.data_ptr() % 256 == 0
    return buf, buf.as_strided(shape, strides, offset)


def _only_there(buf, view):
    """Nothing but the view's elements was written."""
    seen = torch.zeros(buf.shape, dtype=torch.bool, device="cuda")
    seen.as_strided(view.shape, view.stride(), view.storage_offset()).fill_(True)
    return bool((buf[~seen] == 7).all())


def _ptr(t):
    return t.data_ptr()


def _workspace(args, backward):
    n = _lib.load().attn_bwd_b200_fused_workspace(ctypes.byref(args), backward)
    assert n >= 0
    return torch.empty(max(n, 1), dtype=torch.uint8, device="cuda"), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64)])
@pytest.mark.parametrize("heads,kv,sq", [(6, 2, 20), (4, 4, 150)])   # rows of a group in one tile, and rows of a head
@pytest.mark.parametrize("offset", [0, 8, 16, 24])
def test_outputs_at_any_16_bytes(cuda, offset, heads, kv, sq, dtype, d):
    q, k, v, _ = _inputs(2, heads, kv, sq, sq, d, dtype)
    want, wl = ab.fused_attn_fwd(q, k, v, causal=True)
    c = ab.fused._Call(q, k, v, None, 0.0, None, True, None, None)
    buf, o = _place(want.shape, want.stride(), offset, dtype)
    lse = torch.empty_like(wl)
    ws, n = _workspace(c.args, 0)
    _lib.call("attn_bwd_b200_fused_fwd", ctypes.byref(c.args), _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse), _ptr(ws), n,
              torch.cuda.current_stream().cuda_stream)
    assert torch.equal(o, want) and torch.equal(lse, wl) and _only_there(buf, o)
    assert ab.poll_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64)])
@pytest.mark.parametrize("bs,kv", [(20, 4), (1, 2)])   # key tiles that write their results, and parts that are joined
@pytest.mark.parametrize("offset,row,gap", [(8, 0, 0), (0, 8, 0), (0, 0, 8), (16, 16, 16), (24, 24, 40)])
def test_gradients_at_any_16_bytes(cuda, offset, row, gap, bs, kv, dtype, d):
    """Gradients whose rows lie d + row elements apart and whose heads leave a gap."""
    q, k, v, do = _inputs(bs, 2 * kv, kv, 90, 130, d, dtype)
    o, lse = ab.fused_attn_fwd(q, k, v, causal=True)
    want = ab.fused_attn_bwd(do, q, k, v, o, lse, causal=True)
    c = ab.fused._Call(q, k, v, None, 0.0, None, True, None, None)
    bufs, grads = [], []
    for t, dst in zip(want, (c.args.dq_stride, c.args.dk_stride, c.args.dv_stride)):
        b, h, s, _ = t.shape
        head = s * (d + row) + gap
        buf, g = _place(t.shape, (h * head + gap, head, d + row, 1), offset, dtype)
        dst[:] = g.stride()[:3]
        bufs.append(buf)
        grads.append(g)
    ws, n = _workspace(c.args, 1)
    _lib.call("attn_bwd_b200_fused_bwd", ctypes.byref(c.args), _ptr(do), _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse),
              *[_ptr(g) for g in grads], _ptr(ws), n, torch.cuda.current_stream().cuda_stream)
    for buf, g, w in zip(bufs, grads, want):
        assert torch.equal(g, w) and _only_there(buf, g)
    assert ab.poll_error() == 0


def test_documents_of_no_queries_without_device():
    """An array of no elements has no address."""
    from test_fused import _args
    lib, a = _lib.load(), _args(seq_q=0, kv_documents=16)
    assert lib.attn_bwd_b200_fused_fwd(ctypes.byref(a), 0, 16, 16, 0, 0, 0, 0, 0) == _lib.OK
    a = _args(seq_q=0, seq_kv=0, q_documents=16)
    assert lib.attn_bwd_b200_fused_bwd(ctypes.byref(a), *[0] * 9, 0, 0, 0) == _lib.OK
    a = _args(bs=0, q_documents=16)
    assert lib.attn_bwd_b200_fused_bwd(ctypes.byref(a), *[0] * 9, 0, 0, 0) == _lib.OK
    for kw in (dict(kv_documents=16), dict(seq_kv=0, kv_documents=16), dict(q_documents=16)):
        assert lib.attn_bwd_b200_fused_fwd(ctypes.byref(_args(**kw)), 16, 16, 16, 16, 16, 0, 0, 0) == _lib.EINVAL


@pytest.mark.gpu
@pytest.mark.parametrize("bs,sq,skv", [(2, 5, 0), (2, 0, 5), (2, 0, 0), (0, 3, 4), (1, 1, 0), (3, 200, 0), (3, 0, 200)])
@pytest.mark.parametrize("causal", [False, True])
def test_documents_of_no_positions(cuda, bs, sq, skv, causal):
    q, k, v, do = _inputs(bs, 4, 2, sq, skv, 64, BF)
    docs = tuple(torch.zeros(bs, n, dtype=torch.int32, device="cuda") for n in (sq, skv))
    o, lse = ab.fused_attn_fwd(q, k, v, documents=docs, causal=causal, softcap=5.0)
    dq, dk, dv = ab.fused_attn_bwd(do, q, k, v, o, lse, documents=docs, causal=causal, softcap=5.0)
    assert o.shape == (bs, sq, 4, 64) and (o == 0).all() and (lse == -float("inf")).all()
    for g, t in ((dq, q), (dk, k), (dv, v)):
        assert g.shape == t.shape and (g == 0).all()
    assert ab.poll_error() == 0


def test_backward_over_more_keys_than_a_unit_may_have():
    """A unit of dq runs over all keys; its kernel's waits end after 2 s."""
    from test_fused import _args
    lib = _lib.load()
    for keys, code in (((1 << 25) + 1, _lib.EUNSUPPORTED), ((1 << 30) - 1, _lib.EUNSUPPORTED)):
        assert lib.attn_bwd_b200_fused_bwd(ctypes.byref(_args(seq_kv=keys)), *[16] * 9, 0, 0, 0) == code


@pytest.mark.gpu
def test_units_stay_below_the_waits_limit(cuda):
    """Enough rows for every SM, and so no split for their sake: long axes are split all the same."""
    from test_fused import _args
    lib = _lib.load()
    need = lambda back, **kw: lib.attn_bwd_b200_fused_workspace(ctypes.byref(_args(bs=300, heads=1, kv_heads=1, **kw)), back)
    part = 300 * 4 * 129   # one part: fp32 outputs and statistics of a row, 128 elements a head
    assert need(0, seq_q=1, seq_kv=1 << 25) == 2 * part          # two chains of one CTA
    assert need(0, seq_q=1, seq_kv=(1 << 25) + 1) == 4 * part
    assert need(0, seq_q=300, seq_kv=1 << 25) == 0
    assert need(0, seq_q=300, seq_kv=1 << 27) == 300 * 4 * part
    stat = lambda n: 2 * 300 * n * 4
    assert need(1, seq_q=1 << 25, seq_kv=8) == stat(1 << 25)
    assert need(1, seq_q=1 << 26, seq_kv=8) == stat(1 << 26) + 2 * 300 * 8 * 2 * 128 * 4
