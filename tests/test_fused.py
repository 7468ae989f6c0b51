"""Fused attention with capped, biased and masked scores: the 64-bit reference against differences
(CPU), refusals (CPU), and the kernels against the reference (GPU)."""
import ctypes
import math

import pytest
import torch

import attn_bwd_b200 as ab
from attn_bwd_b200 import _lib
from fused_reference import attention, seen

BF, HF = torch.bfloat16, torch.float16


# ------------------------------------------------------------------ the reference itself
@pytest.mark.parametrize("mods", [dict(), dict(causal=True), dict(softcap=3.0), dict(slopes=[0.5, 0.1]),
                                  dict(causal=True, prefix_lens=[4], softcap=2.0, slopes=[0.2, 0.0]),
                                  dict(causal=True, documents=[[0, 0, 0, 1, 1, 2, -1]])])
def test_reference_gradients_against_differences(mods):
    torch.manual_seed(0)
    mods = dict(mods)
    if "documents" in mods:
        mods["documents"] = torch.tensor(mods["documents"])
    q, k, v, do = (torch.randn(s, dtype=torch.float64) for s in ((1, 2, 7, 4), (1, 1, 7, 4), (1, 1, 7, 4), (1, 7, 2, 4)))
    loss = lambda q, k, v: float((attention(q, k, v, half=0.0, **mods)["o"] * do).sum())
    r = attention(q, k, v, do, half=0.0, **mods)
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        step = torch.randn_like(x)
        up = [x + 1e-5 * step if y is x else y for y in (q, k, v)]
        dn = [x - 1e-5 * step if y is x else y for y in (q, k, v)]
        diff = (loss(*up) - loss(*dn)) / 2e-5
        assert abs(diff - float((r[name] * step).sum())) < 1e-6 * (1 + abs(diff))


# ------------------------------------------------------------------ refusals
def _cpu(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def test_cpu_tensors_are_refused():
    q, k = _cpu(1, 8, 4, 128), _cpu(1, 2, 4, 128)
    with pytest.raises(ValueError, match="CUDA"):
        ab.fused_attn_fwd(q, k, k)
    with pytest.raises(ValueError, match="CUDA"):
        ab.fused_attn_bwd(q.transpose(1, 2), q, k, k, q.transpose(1, 2), torch.zeros(1, 8, 4))
    with pytest.raises(TypeError):
        ab.fused_attn_fwd(None, k, k)


def _args(**kw):
    a = _lib.FusedArgs()
    base = dict(bs=1, seq_q=4, seq_kv=4, heads=8, kv_heads=2, head_dim=128, dtype=0, causal=0, scale=0.1, softcap=0.0)
    base.update(kw)
    for n, x in base.items():
        setattr(a, n, x)
    for f, h in (("q_stride", a.heads), ("k_stride", a.kv_heads), ("v_stride", a.kv_heads), ("dq_stride", a.heads),
                 ("dk_stride", a.kv_heads), ("dv_stride", a.kv_heads)):
        getattr(a, f)[:] = (max(1, h) * 4 * 128, 4 * 128, 128)
    return a


@pytest.mark.parametrize("bad,code", [
    (dict(bs=-1), _lib.EINVAL), (dict(seq_q=-1), _lib.EINVAL), (dict(seq_kv=-4), _lib.EINVAL), (dict(heads=0), _lib.EINVAL),
    (dict(kv_heads=3), _lib.EINVAL), (dict(scale=0.0), _lib.EINVAL), (dict(scale=-1.0), _lib.EINVAL),
    (dict(scale=math.nan), _lib.EINVAL), (dict(scale=math.inf), _lib.EINVAL), (dict(softcap=-1.0), _lib.EINVAL),
    (dict(softcap=math.nan), _lib.EINVAL), (dict(softcap=1e-35), _lib.EINVAL), (dict(scale=3e38), _lib.EINVAL),
    (dict(scale=1e10, softcap=1e-25), _lib.EINVAL), (dict(head_dim=96), _lib.EUNSUPPORTED), (dict(dtype=2), _lib.EUNSUPPORTED),
    (dict(prefix_lens=16), _lib.EINVAL), (dict(q_documents=16), _lib.EINVAL), (dict(kv_documents=16), _lib.EINVAL),
    (dict(bs=70000), _lib.EINVAL), (dict(seq_q=1 << 30), _lib.EINVAL)])
def test_c_entry_refuses_without_device(bad, code):
    lib, a = _lib.load(), _args(**bad)
    p = ctypes.byref(a)
    assert lib.attn_bwd_b200_fused_fwd(p, 16, 16, 16, 16, 16, 0, 0, 0) == code
    assert lib.attn_bwd_b200_fused_bwd(p, *[16] * 9, 0, 0, 0) == code
    assert lib.attn_bwd_b200_fused_workspace(p, 0) == -code


def test_c_entry_refuses_pointers_and_strides_without_device():
    lib, a = _lib.load(), _args()
    p = ctypes.byref(a)
    assert lib.attn_bwd_b200_fused_fwd(None, 16, 16, 16, 16, 16, 0, 0, 0) == _lib.EINVAL
    assert lib.attn_bwd_b200_fused_fwd(p, 0, 16, 16, 16, 16, 0, 0, 0) == _lib.EINVAL
    assert lib.attn_bwd_b200_fused_fwd(p, 16, 24, 16, 16, 16, 0, 0, 0) == _lib.EALIGN
    assert lib.attn_bwd_b200_fused_bwd(p, *[16] * 6, 0, 16, 16, 0, 0, 0) == _lib.EINVAL
    for f in ("q_stride", "k_stride", "v_stride"):
        a = _args()
        getattr(a, f)[2] = 129
        assert lib.attn_bwd_b200_fused_fwd(ctypes.byref(a), 16, 16, 16, 16, 16, 0, 0, 0) == _lib.EALIGN
        getattr(a, f)[2] = 0
        assert lib.attn_bwd_b200_fused_fwd(ctypes.byref(a), 16, 16, 16, 16, 16, 0, 0, 0) == _lib.EALIGN
    a = _args(seq_q=(2048 << 7) + 1, q_documents=16, kv_documents=16)   # more tiles than a list of documents holds
    assert lib.attn_bwd_b200_fused_bwd(ctypes.byref(a), *[16] * 9, 0, 0, 0) == _lib.EUNSUPPORTED
    a = _args(bs=0)   # nothing to do
    assert lib.attn_bwd_b200_fused_fwd(ctypes.byref(a), 0, 0, 0, 0, 0, 0, 0, 0) == _lib.OK
    assert lib.attn_bwd_b200_fused_bwd(ctypes.byref(a), *[0] * 9, 0, 0, 0) == _lib.OK


@pytest.mark.gpu
def test_python_refusals(cuda):
    q, k = _cpu(1, 8, 4, 128).cuda(), _cpu(1, 2, 4, 128).cuda()
    bad = [dict(scale=0.0), dict(scale=-1.0), dict(softcap=-2.0), dict(softcap=math.inf),
           dict(prefix_lens=torch.zeros(1, dtype=torch.int32, device="cuda")),
           dict(slopes=torch.zeros(7, device="cuda")), dict(documents=torch.zeros(1, 5, dtype=torch.int32, device="cuda"))]
    for kw in bad:
        with pytest.raises(ValueError):
            ab.fused_attn_fwd(q, k, k, **kw)
    for kw in [dict(slopes=torch.zeros(8, device="cuda").double()),
               dict(documents=torch.zeros(1, 4, dtype=torch.int64, device="cuda"))]:
        with pytest.raises(TypeError):
            ab.fused_attn_fwd(q, k, k, **kw)
    with pytest.raises(TypeError):
        ab.fused_attn_fwd(q.float(), k.float(), k.float())
    with pytest.raises(TypeError):
        ab.fused_attn_fwd(q, k.half(), k)
    for qq, kk in ((q, k[..., :64]), (q[:, :7], k), (q[..., :96], k[..., :96]), (q, k.expand(2, -1, -1, -1))):
        with pytest.raises(ValueError):
            ab.fused_attn_fwd(qq, kk, kk)
    with pytest.raises(ValueError, match="pair"):
        ab.fused_attn_fwd(q, torch.cat([k, k], 2), torch.cat([k, k], 2),
                          documents=torch.zeros(1, 4, dtype=torch.int32, device="cuda"))
    o, lse = ab.fused_attn_fwd(q, k, k)
    for args in ((o[:, :3], q, k, k, o, lse), (o, q, k, k, o, lse[:, :, :3]), (o, q, k, k, o.transpose(1, 2), lse)):
        with pytest.raises(ValueError):
            ab.fused_attn_bwd(*args)


# ------------------------------------------------------------------ the kernels
def _inputs(bs, h, kv, sq, skv, d, dtype, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g)
    q, k, v = mk(bs, h, sq, d) * std, mk(bs, kv, skv, d), mk(bs, kv, skv, d)
    return [t.to(dtype).cuda() for t in (q, k, v, mk(bs, sq, h, d))]


def _docs(bs, n, mean, seed=0, pad=0, start=0):
    g = torch.Generator().manual_seed(seed)
    rows = []
    for _ in range(bs):
        row, d = [], start
        while len(row) < n - pad:
            row += [d] * int(torch.randint(1, 2 * mean, (1,), generator=g))
            d += 1
        rows.append(row[:n - pad] + [-1] * pad)
    return torch.tensor(rows, dtype=torch.int32)


def _within(got, ref, tol, name):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, name
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]), name
    err = (got[~inf] - ref[~inf]).abs()
    assert torch.isfinite(err).all(), f"{name}: not finite"
    over = err - tol[~inf]
    assert not (over > 0).any(), f"{name}: over the bound by {float(over.max()):.3g} (error {float(err.max()):.3g})"


def _check(q, k, v, do, back=True, **mods):
    o, lse = ab.fused_attn_fwd(q, k, v, **mods)
    r = attention(q, k, v, do if back else None, **mods)
    _within(o, r["o"], r["o_tol"], "o")
    _within(lse, r["lse"], r["lse_tol"], "lse")
    if back:
        grads = ab.fused_attn_bwd(do, q, k, v, o, lse, **mods)
        for g, n in zip(grads, ("dq", "dk", "dv")):
            _within(g, r[n], r[n + "_tol"], n)
    assert ab.poll_error() == 0
    return o, lse


SIZES = [(1, 1, 1), (1, 1, 129), (2, 127, 127), (1, 128, 128), (1, 129, 257), (2, 64, 96), (1, 301, 467), (1, 300, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64)])
@pytest.mark.parametrize("heads,kv", [(1, 1), (6, 2), (10, 1), (4, 4)])
@pytest.mark.parametrize("bs,sq,skv", SIZES)
@pytest.mark.parametrize("causal", [False, True])
def test_sizes_and_heads(cuda, bs, sq, skv, causal, heads, kv, dtype, d):
    _check(*_inputs(bs, heads, kv, sq, skv, d, dtype), causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(HF, 128), (BF, 64)])
@pytest.mark.parametrize("bs,sq,skv", SIZES)
@pytest.mark.parametrize("mod", ["cap", "slopes", "prefix", "docs", "all"])
def test_modified_scores(cuda, mod, bs, sq, skv, dtype, d):
    q, k, v, do = _inputs(bs, 6, 2, sq, skv, d, dtype, std=3.0)
    kw = {}
    if mod in ("cap", "all"):
        kw["softcap"] = 5.0
    if mod in ("slopes", "all"):
        kw["slopes"] = torch.tensor([0.5, 0.25, 0.125, 0.0, 0.03, 1.0]).cuda()
    if mod in ("prefix", "all"):
        kw["prefix_lens"] = torch.tensor([skv // 2, 0][:bs], dtype=torch.int32).cuda()
        kw["causal"] = True
    if mod in ("docs", "all"):
        kd = _docs(bs, skv, max(2, skv // 3), pad=skv // 10)
        qd = torch.cat([torch.full((bs, max(0, sq - skv)), -1, dtype=torch.int32), kd], 1)[:, -sq:]
        kw["documents"] = (qd.contiguous().cuda(), kd.cuda())
    _check(q, k, v, do, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("std,kw", [
    (1.0, dict(softcap=1e-4)), (1.0, dict(softcap=1e8)), (1.0, dict(softcap=1e30)), (8.0, dict(softcap=2.0)),
    (1.0, dict(scale=1e-30)), (1.0, dict(scale=4.0)), (0.0, dict(softcap=1e-20)), (20.0, dict(softcap=50.0))])
def test_extreme_caps_and_scales(cuda, std, kw):
    """Caps far above and below the scores, scores at the cap, scales that leave nothing of them."""
    q, k, v, do = _inputs(1, 4, 2, 150, 260, 64, BF, std=std)
    _check(q, k, v, do, causal=True, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 3, 5])
def test_tokens_over_few_and_odd_tiles(cuda, n):
    """One tile of rows: two chains over alternate key tiles, the last of them odd; with documents too."""
    skv = n * 128 - 7
    q, k, v, do = _inputs(3, 8, 2, 4, skv, 64, HF)
    _check(q, k, v, do, causal=True)
    kd = _docs(3, skv, 90, pad=3)
    _check(q, k, v, do, causal=True, documents=(kd[:, -4:].contiguous().cuda(), kd.cuda()), softcap=3.0)


@pytest.mark.gpu
def test_many_short_units(cuda):
    """More units than SMs, most of them of one tile, some of none: each CTA takes up several."""
    q, k, v, do = _inputs(24, 12, 4, 130, 70, 64, BF)
    _check(q, k, v, do, causal=True)
    kd = _docs(24, 130, 20, pad=30)
    q, k, v, do = _inputs(24, 12, 4, 130, 130, 64, BF)
    _check(q, k, v, do, causal=True, documents=kd.cuda())


@pytest.mark.gpu
def test_one_head_for_many(cuda):
    _check(*_inputs(1, 128, 1, 3, 200, 64, BF), causal=True)     # a position's heads fill a tile
    _check(*_inputs(1, 160, 1, 2, 70, 64, BF), causal=True)      # more heads than a tile has rows
    _check(*_inputs(1, 80, 8, 40, 130, 128, BF), causal=True)    # the layer's own head layout


@pytest.mark.gpu
def test_unordered_documents_and_masks_that_leave_rows_empty(cuda):
    q, k, v, do = _inputs(2, 4, 2, 270, 300, 64, BF)
    g = torch.Generator().manual_seed(3)
    kd = torch.randint(-1, 4, (2, 300), generator=g, dtype=torch.int32).cuda()
    qd = torch.randint(-1, 6, (2, 270), generator=g, dtype=torch.int32).cuda()   # 4 and 5 have no keys
    for causal in (False, True):
        o, lse = _check(q, k, v, do, documents=(qd, kd), causal=causal)
        none = (qd < 0) | (qd > 3)
        assert none.any() and torch.isinf(lse.transpose(1, 2)[none]).all() and (o[none] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 128), (BF, 64), (HF, 64)])
@pytest.mark.parametrize("mods", [{}, {"softcap": 15.0}, {"softcap": 1e5}, {"slopes": True}, {"softcap": 4.0, "slopes": True},
                                  {"documents": True}])
@pytest.mark.parametrize("sq,skv", [(8, 8), (1, 128), (100, 100), (64, 96), (256, 100)])
def test_gradients_of_few_keys(cuda, sq, skv, mods, dtype, d):
    """Rows of one, two, three keys, where ds is small beside what the output's rounding does to delta."""
    q, k, v, do = _inputs(2, 4, 2, sq, skv, d, dtype, seed=sq, std=3.0)
    mods = dict(mods, causal=True)
    if "slopes" in mods:
        mods["slopes"] = torch.tensor([0.5, 0.25, 0.03, 1.0], device="cuda")
    if "documents" in mods:
        docs = _docs(2, max(sq, skv), 5, pad=3).cuda()
        mods["documents"] = (docs[:, -sq:].contiguous(), docs[:, -skv:].contiguous())
    o, lse = ab.fused_attn_fwd(q, k, v, **mods)
    r = attention(q, k, v, do, one_tile=True, **mods)
    for g, n in zip(ab.fused_attn_bwd(do, q, k, v, o, lse, **mods), ("dq", "dk", "dv")):
        _within(g, r[n], r[n + "_tol"], n)


@pytest.mark.gpu
def test_nothing_to_see(cuda):
    q, k, v, do = _inputs(1, 4, 2, 5, 0, 128, BF)
    o, lse = _check(q, k, v, do)
    assert (o == 0).all() and (lse == -math.inf).all()
    q, k, v, do = _inputs(1, 4, 2, 0, 9, 128, BF)
    o, lse = ab.fused_attn_fwd(q, k, v)
    dq, dk, dv = ab.fused_attn_bwd(do, q, k, v, o, lse)
    assert o.shape == (1, 0, 4, 128) and dq.shape == q.shape and (dk == 0).all() and (dv == 0).all()
    q, k, v, do = _inputs(0, 4, 2, 3, 9, 128, BF)
    o, lse = ab.fused_attn_fwd(q, k, v)
    assert o.shape == (0, 3, 4, 128) and ab.fused_attn_bwd(do, q, k, v, o, lse)[1].shape == k.shape


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_padding_holds_anything(cuda, bad):
    """Queries and keys of no document (behind the last one, and between documents) reach nothing."""
    q, k, v, do = _inputs(2, 4, 2, 300, 300, 128, BF)
    docs = _docs(2, 300, 60, pad=45)
    docs[0, 100:133] = -1
    pad = (docs < 0).cuda()
    for t in (q, k, v):
        t.transpose(1, 2)[pad] = bad
    do[pad] = bad
    for causal in (False, True):
        o, lse = _check(q, k, v, do, documents=docs.cuda(), causal=causal)
        assert (o[pad] == 0).all()


@pytest.mark.gpu
def test_future_scores_of_any_size_reach_nothing(cuda):
    """Keys behind the diagonal whose scores are the type's largest values."""
    q, k, v, do = _inputs(1, 2, 1, 200, 200, 64, HF)
    k[:, :, 150:] = 60000.0
    r = attention(q[:, :, :150], k[:, :, :150], v[:, :, :150], causal=True)
    o, lse = ab.fused_attn_fwd(q, k, v, causal=True)
    _within(o[:, :150], r["o"], r["o_tol"], "o")


@pytest.mark.gpu
@pytest.mark.parametrize("sq,skv,heads,kv,docs", [(1, 5000, 10, 1, False), (1, 4097, 4, 4, False), (7, 3001, 6, 2, False),
                                                   (3, 2000, 6, 2, True), (40, 2100, 10, 2, False)])
def test_split_keys(cuda, sq, skv, heads, kv, docs):
    """Few queries over many keys: the keys are shared among CTAs and the parts joined."""
    q, k, v, do = _inputs(2, heads, kv, sq, skv, 128, BF)
    kw = {}
    if docs:   # the first row's queries see the last keys only, the second row's nothing
        kd = torch.zeros(2, skv, dtype=torch.int32)
        kd[0, -30:] = 1
        qd = torch.tensor([[1] * sq, [7] * sq], dtype=torch.int32)
        kw["documents"] = (qd.cuda(), kd.cuda())
    _check(q, k, v, do, causal=True, **kw)


@pytest.mark.gpu
def test_strides(cuda):
    """Heads inside positions, a slice of a longer cache, every other position, and layouts that
    have to be copied (unaligned rows, a broadcast batch): the same results, gradients shaped alike."""
    q, k, v, do = _inputs(2, 6, 2, 140, 200, 64, BF)
    mods = dict(causal=True)
    o, lse = ab.fused_attn_fwd(q, k, v, **mods)
    grads = ab.fused_attn_bwd(do, q, k, v, o, lse, **mods)

    def same(q2, k2, v2, do2=do):
        o2, lse2 = ab.fused_attn_fwd(q2, k2, v2, **mods)
        assert torch.equal(o2, o) and torch.equal(lse2, lse)
        for x, y, like in zip(ab.fused_attn_bwd(do2, q2, k2, v2, o2, lse2, **mods), grads, (q2, k2, v2)):
            assert torch.equal(x, y) and x.shape == like.shape

    bshd = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    same(bshd(q), bshd(k), v)
    cache = torch.full((2, 2, 500, 64), math.nan, dtype=BF, device="cuda")
    cache[:, :, 300:] = k
    same(q, cache[:, :, 300:], bshd(v))
    twice = torch.full((2, 2, 400, 64), math.nan, dtype=BF, device="cuda")
    twice[:, :, ::2] = v
    same(q, k, twice[:, :, ::2])
    wide = torch.zeros(2, 6, 140, 67, dtype=BF, device="cuda")[..., 3:]
    wide.copy_(q)
    same(wide, k, v)
    same(q, k, v, do.transpose(0, 1).contiguous().transpose(0, 1))
    k1 = k[:1].expand(2, -1, -1, -1)
    o3, _ = ab.fused_attn_fwd(q, k1, v, **mods)
    assert torch.equal(o3, ab.fused_attn_fwd(q, k1.contiguous(), v, **mods)[0])


@pytest.mark.gpu
def test_equal_bits_and_graph_replay(cuda):
    """Equal inputs give equal bits (kernels, splits, replays), on another stream too."""
    q, k, v, do = _inputs(1, 10, 1, 200, 700, 128, BF)
    mods = dict(causal=True, softcap=20.0)
    o, lse = ab.fused_attn_fwd(q, k, v, **mods)
    grads = ab.fused_attn_bwd(do, q, k, v, o, lse, **mods)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        o2, lse2 = ab.fused_attn_fwd(q, k, v, **mods)
        g2 = ab.fused_attn_bwd(do, q, k, v, o2, lse2, **mods)
    side.synchronize()
    assert torch.equal(o, o2) and all(torch.equal(a, b) for a, b in zip(grads, g2))
    sq = torch.empty_like(q).copy_(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go, gl = ab.fused_attn_fwd(sq, k, v, **mods)
        gg = ab.fused_attn_bwd(do, sq, k, v, go, gl, **mods)
    q3 = _inputs(1, 10, 1, 200, 700, 128, BF, seed=9)[0]
    for x in (q3, q):
        sq.copy_(x)
        graph.replay()
        e, el = ab.fused_attn_fwd(x, k, v, **mods)
        eg = ab.fused_attn_bwd(do, x, k, v, e, el, **mods)
        assert torch.equal(go, e) and torch.equal(gl, el) and all(torch.equal(a, b) for a, b in zip(gg, eg))
    assert ab.poll_error() == 0


@pytest.mark.gpu
def test_documents_change_between_replays(cuda):
    """A captured training pass over documents reads their numbers, prefixes and slopes at each replay."""
    q, k, v, do = _inputs(2, 4, 2, 300, 300, 64, HF)
    docs = [_docs(2, 300, m, seed=m, pad=p).cuda() for m, p in ((40, 0), (90, 37), (300, 5), (10, 299))]
    pre = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 200], [70, 300], [0, 0], [5, 1])]
    d, p, sl = docs[0].clone(), pre[0].clone(), torch.tensor([0.5, 0.1, 0.02, 0.0], device="cuda")
    mods = dict(causal=True, documents=d, prefix_lens=p, slopes=sl)

    def step():
        o, lse = ab.fused_attn_fwd(q, k, v, **mods)
        t, tl = ab.fused_attn_fwd(q[:, :, -1:], k, v, causal=True, documents=(d[:, -1:].contiguous(), d))
        return (o, lse, t, tl) + ab.fused_attn_bwd(do, q, k, v, o, lse, **mods)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for x, y in zip(docs + docs[:1], pre + pre[:1]):
        d.copy_(x)
        p.copy_(y)
        graph.replay()
        held = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(held, step()))
    assert ab.poll_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("docs", [False, True])
def test_calls_close_behind_one_another(cuda, docs):
    """Calls that take the last one's workspace at once (kernels of a call overlap, calls do not)."""
    sets = [_inputs(1, 10, 1, 3, 2000, 128, BF, seed=s) for s in range(4)]
    ids = [_docs(1, 2000, 50 + 400 * s, seed=s).cuda() for s in range(4)]

    def step(i):
        q, k, v, do = sets[i]
        mods = dict(causal=True, documents=(ids[i][:, -3:].contiguous(), ids[i])) if docs else dict(causal=True)
        o, lse = ab.fused_attn_fwd(q, k, v, **mods)
        return (o, lse) + ab.fused_attn_bwd(do, q, k, v, o, lse, **mods)

    alone = []
    for i in range(4):
        alone.append(step(i))
        torch.cuda.synchronize()
    runs = [step(i % 4) for i in range(64)]
    for i, r in enumerate(runs):
        assert all(torch.equal(a, b) for a, b in zip(alone[i % 4], r)), i
    assert ab.poll_error() == 0


@pytest.mark.gpu
def test_layer_step_with_rope(cuda):
    """The operators as a training step calls them: rotate, attend, and back through both; the
    gradients of the unrotated queries and keys against the formulas'."""
    from fused_reference import rope
    bs, s, h, kv, d = 2, 150, 10, 2, 128
    q, k, v, do = _inputs(bs, h, kv, s, s, d, BF, seed=4)
    table = ab.rope_table(d)
    pos = torch.arange(s, device="cuda")
    qr, kr = ab.rope_fwd(q, k, pos, table)
    o, lse = ab.fused_attn_fwd(qr, kr, v, causal=True)
    dqr, dkr, dv = ab.fused_attn_bwd(do, qr, kr, v, o, lse, causal=True)
    dq, dk = ab.rope_bwd(dqr, dkr, pos, table)
    r = attention(qr, kr, v, do, causal=True)
    f = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    for got, n in ((dq, "dq"), (dk, "dk")):
        want = rope(r[n], pos.cpu(), f, d, inverse=True)
        # a rotation mixes the errors of a pair's two elements; one more rounding
        t = r[n + "_tol"]
        t = t + torch.cat([t[..., d // 2:], t[..., :d // 2]], -1) + 2 ** -8 * want.abs() + 1e-7
        _within(got, want, t, n)
    _within(dv, r["dv"], r["dv_tol"], "dv")


@pytest.mark.gpu
def test_agrees_with_the_materialised_backward(cuda):
    """The layer's head layout, no dropout: dv and the gradient of the scores of the path that is given
    the weights belong to the same function (dq = scale * dS k, sum over its own dS)."""
    bs, sq, skv = 1, 96, 112
    q, k, v, do = _inputs(bs, 80, 8, sq, skv, 128, BF, seed=6)
    o, lse = ab.fused_attn_fwd(q, k, v)
    dq, dk, dv = ab.fused_attn_bwd(do, q, k, v, o, lse)
    scores = torch.matmul(q.double(), k.double().repeat_interleave(10, 1).transpose(2, 3)) / math.sqrt(128)
    P = torch.softmax(scores, -1).to(BF)
    dS, dV = ab.custom_kernel((do, P, P, v, torch.ones_like(P, dtype=torch.bool), 0.0))
    r = attention(q, k, v, do)
    # P rounded to bf16 enters the other path as an input, like this path's own rounding of it
    assert ((dV.double() - dv.double()).abs().cpu() <= 2.2 * r["dv_tol"]).all()
    dq2 = torch.matmul(dS.double(), k.double().repeat_interleave(10, 1)) / math.sqrt(128)
    assert (dq2.cpu() - dq.double().cpu()).norm() <= 2 ** -7 * dq2.norm().cpu()


@pytest.mark.gpu
def test_workspace_is_checked(cuda):
    q, k, v, do = _inputs(1, 4, 1, 1, 2000, 128, BF)
    c = ab.fused._Call(q, k, v, None, 0.0, None, True, None, None)
    need = _lib.load().attn_bwd_b200_fused_workspace(ctypes.byref(c.args), 0)
    assert need > 0
    o, lse = torch.empty(1, 1, 4, 128, dtype=BF, device="cuda"), torch.empty(1, 4, 1, device="cuda")
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    call = lambda w, n: _lib.load().attn_bwd_b200_fused_fwd(ctypes.byref(c.args), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                                            o.data_ptr(), lse.data_ptr(), w, n, 0)
    assert call(0, 0) == _lib.EINVAL and call(ws.data_ptr(), need - 1) == _lib.EINVAL
    assert call(ws.data_ptr() + 16, need) == _lib.EALIGN
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_two_streams_at_once(cuda):
    """Calls that overlap on two streams, each with its own workspace, give the bits they give alone."""
    sets = [_inputs(2, 10, 2, 300, 900, 128, BF, seed=s) for s in (1, 2)]
    mods = dict(causal=True, softcap=15.0)

    def step(q, k, v, do):
        o, lse = ab.fused_attn_fwd(q, k, v, **mods)
        t, tl = ab.fused_attn_fwd(q[:, :, -1:], k, v, **mods)
        return (o, lse, t, tl) + ab.fused_attn_bwd(do, q, k, v, o, lse, **mods)

    alone = [step(*x) for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(step(*sets[i]))
    torch.cuda.synchronize()
    for a, runs in zip(alone, got):
        assert all(torch.equal(x, y) for r in runs for x, y in zip(a, r))
    assert ab.poll_error() == 0


@pytest.mark.gpu
def test_long_cache(cuda):
    """17 million keys: element offsets above 2^31.  A few planted keys, the last one among them, take
    nearly all of the weight; the rest is noise of known size."""
    n, d = 17_000_003, 128
    g = torch.Generator(device="cuda").manual_seed(0)
    k = torch.empty(1, 1, n, d, dtype=BF, device="cuda").normal_(generator=g).mul_(0.01)
    v = torch.empty(1, 1, n, d, dtype=BF, device="cuda").normal_(generator=g)
    q = torch.randn(1, 4, 1, d, generator=g, device="cuda").to(BF)
    at = [5, 8_388_607, 16_777_216, 16_900_000, n - 1]
    for a, h in zip(at, (0, 1, 2, 3, 0)):
        k[0, 0, a] = q[0, h, 0] * 3        # score about 3 * 128 / sqrt(128) = 34 for its head
    o, lse = ab.fused_attn_fwd(q, k, v, causal=True)
    ref, rl = torch.zeros(4, d, dtype=torch.float64, device="cuda"), torch.full((4, 1), -math.inf, device="cuda").double()
    for c in range(0, n, 1 << 21):
        s = q[0, :, 0].double() @ k[0, 0, c:c + (1 << 21)].double().t() / math.sqrt(d)
        part = torch.logsumexp(s, 1, keepdim=True)
        new = torch.logaddexp(rl, part)
        ref = ref * torch.exp(rl - new) + torch.exp(s - new) @ v[0, 0, c:c + (1 << 21)].double()
        rl = new
    # weights rounded to bf16 and the result once: 2 half steps of values up to 5, and fp32 sums
    assert (o[0, 0].double() - ref).abs().max() < 2 * 2 ** -8 * 5
    assert ref.abs().max() > 0.5           # the planted keys, not the mean of the noise
    assert (lse[0].double() - rl).abs().max() < 1e-4


@pytest.mark.gpu
def test_cache_slices_far_from_its_start(cuda):
    """Keys and values that lie above 2^32 bytes in their buffer, gradients in their own."""
    big = torch.zeros(2, 2, 4_400_000, 128, dtype=BF, device="cuda")    # 4.5 GB a buffer
    q, k, v, do = _inputs(2, 4, 2, 90, 200, 128, BF)
    far = big[:, :, -200:]
    far.copy_(k)
    o, lse = ab.fused_attn_fwd(q, far, v, causal=True)
    e, el = ab.fused_attn_fwd(q, k, v, causal=True)
    assert torch.equal(o, e) and torch.equal(lse, el)
    for a, b in zip(ab.fused_attn_bwd(do, q, far, v, o, lse, causal=True), ab.fused_attn_bwd(do, q, k, v, e, el, causal=True)):
        assert torch.equal(a, b)
