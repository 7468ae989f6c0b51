"""Fused attention where a result could leak or vanish: what padding holds, and numbers that are not
finite under a cap."""
import math

import pytest
import torch

import attn_bwd_b200 as ab
from fused_reference import attention
from test_fused import _inputs, _within

BF, HF = torch.bfloat16, torch.float16


def _mods(mod, heads, bs, skv):
    kw = {}
    if "cap" in mod:
        kw["softcap"] = 5.0
    if "slopes" in mod:
        kw["slopes"] = torch.tensor([0.5, 0.25, 0.0, 0.03, 0.125, 1.0][:heads], device="cuda")
    if "prefix" in mod:
        kw["prefix_lens"] = torch.tensor([skv // 2, 3, 0, skv][:bs], dtype=torch.int32, device="cuda")
    if mod != "full":
        kw["causal"] = True
    return kw


# units of one tile, of several tiles, of packed rows, of split keys, and of two chains over the keys
PADDED = [(2, 4, 2, 300, 300), (2, 4, 2, 100, 100), (1, 6, 1, 70, 460), (2, 4, 2, 1, 2000), (2, 6, 2, 4, 1900), (3, 2, 2, 130, 270)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 128), (BF, 64), (HF, 64)])
@pytest.mark.parametrize("mod", ["full", "causal", "cap", "slopes", "cap+slopes", "cap+prefix", "slopes+prefix"])
@pytest.mark.parametrize("bs,heads,kv,sq,skv", PADDED)
def test_padding_changes_no_bit(cuda, bs, heads, kv, sq, skv, mod, dtype, d):
    """Padding behind the last document, between documents and inside one, in queries and keys: whatever
    it holds, the results are the same bits, and those that the formulas give."""
    q, k, v, do = _inputs(bs, heads, kv, sq, skv, d, dtype, seed=skv, std=3.0)
    g = torch.Generator().manual_seed(skv)
    kd = torch.arange(skv, dtype=torch.int32).div(max(1, skv // 3), rounding_mode="floor").repeat(bs, 1)
    kd[torch.rand(bs, skv, generator=g) < 0.1] = -1
    kd[:, skv - 3 - skv // 16:skv - sq if sq < 3 else skv] = -1
    qd = kd[:, skv - sq:].clone()
    if sq < 3:
        qd[:] = 2   # a token that its cache's padding does not touch
    kw = dict(_mods(mod, heads, bs, skv), documents=(qd.cuda(), kd.cuda()))
    qp, kp = (qd < 0).cuda(), (kd < 0).cuda()
    assert kp.any()

    def step(fill):
        for t, p in ((q.transpose(1, 2), qp), (k.transpose(1, 2), kp), (v.transpose(1, 2), kp), (do, qp)):
            t[p] = fill
        o, lse = ab.fused_attn_fwd(q, k, v, **kw)
        return (o, lse) + ab.fused_attn_bwd(do, q, k, v, o, lse, **kw)

    want = step(0.0)
    r = attention(q, k, v, do, **kw)
    # An exponential below 2^-126 may be taken as 0 (steep slopes reach that): p is then off by up to 2^-126, ds
    # by that times |dp - delta| <= 2 max sum|do| max|v| = a, and dq and dk by a times the sums of |k| and |q|
    # times the scale.  The reference's bound counts this for the rounding of ds, not for p.
    a = 2.0 ** -126 * 2 * float(do.abs().double().sum(-1).max()) * float(v.abs().max()) / math.sqrt(d)
    r["dq_tol"] = r["dq_tol"] + a * float(k.abs().double().sum(2).max())
    r["dk_tol"] = r["dk_tol"] + a * float(q.abs().double().sum((1, 2)).max())
    for x, n in zip(want, ("o", "lse", "dq", "dk", "dv")):
        _within(x, r[n], r[n + "_tol"], n)
    for fill in (3.0, 6e4, math.inf, math.nan):
        for x, y, n in zip(step(fill), want, ("o", "lse", "dq", "dk", "dv")):
            assert torch.equal(x, y), f"{n}, padding of {fill}"
    assert ab.poll_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 128), (BF, 64), (HF, 64)])
@pytest.mark.parametrize("mod", ["cap", "cap+slopes", "full"])
@pytest.mark.parametrize("std", [0.01, 8.0])   # scores far below the cap, and at it
@pytest.mark.parametrize("bs,heads,kv,sq,skv", [(1, 2, 1, 300, 300), (1, 2, 2, 100, 100), (1, 4, 1, 3, 700), (2, 6, 2, 60, 300)])
def test_nan_under_a_cap_stays_nan(cuda, bs, heads, kv, sq, skv, std, mod, dtype, d):
    """A NaN query: its row is NaN, output, statistic and gradient, and so are the gradients of the keys
    that it sees; other rows are what they are without it.  A NaN key: every row that sees it is NaN."""
    q, k, v, do = _inputs(bs, heads, kv, sq, skv, d, dtype, seed=7, std=std)
    kw = dict(_mods(mod, heads, bs, skv), softcap=2.0)
    row, h = sq // 2, heads - 1
    r = attention(q, k, v, do, **kw)
    bad = q.clone()
    bad[0, h, row, d // 3] = math.nan
    o, lse = ab.fused_attn_fwd(bad, k, v, **kw)
    assert torch.isnan(o[0, row, h]).all() and torch.isnan(lse[0, h, row])
    rest = torch.ones(bs, sq, heads, dtype=torch.bool)
    rest[0, row, h] = False
    _within(o.cpu()[rest], r["o"][rest], r["o_tol"][rest], "o")
    rt = rest.transpose(1, 2)
    _within(lse.cpu()[rt], r["lse"][rt], r["lse_tol"][rt], "lse")
    dq, dk, dv = ab.fused_attn_bwd(do, bad, k, v, o, lse, **kw)
    assert torch.isnan(dq[0, h, row]).all()
    last = skv if mod == "full" else skv - sq + row + 1   # keys that the row sees
    assert torch.isnan(dv[0, -1, :last]).all() and torch.isnan(dk[0, -1, :last]).all()
    _within(dq.cpu()[rt], r["dq"][rt], r["dq_tol"][rt], "dq")
    key = skv - sq + sq // 3
    bad = k.clone()
    bad[0, 0, key, 1] = math.nan
    o, lse = ab.fused_attn_fwd(q, bad, v, **kw)
    first = 0 if mod == "full" else sq // 3   # rows that see the key
    grp = heads // kv
    assert torch.isnan(o[0, first:, :grp]).all() and torch.isnan(lse[0, :grp, first:]).all()
    dq, dk, dv = ab.fused_attn_bwd(do, q, bad, v, o, lse, **kw)
    assert torch.isnan(dq[0, :grp, first:]).all() and torch.isnan(dv[0, 0, key]).all() and torch.isnan(dk[0, 0, key]).all()
    if kv > 1:   # the other groups
        assert torch.isfinite(o[0, :, grp:]).all() and torch.isfinite(dv[0, 1:]).all()
    assert ab.poll_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [1e-60, 5e-324, 1e-46, 1e-35, 1e-30, -1e-60, math.nan, math.inf])
def test_caps_too_low_to_be_told_from_none_are_refused(cuda, cap):
    q, k, v, do = _inputs(1, 2, 1, 4, 4, 64, BF)
    o, lse = ab.fused_attn_fwd(q, k, v)
    with pytest.raises(ValueError, match="softcap"):
        ab.fused_attn_fwd(q, k, v, softcap=cap)
    with pytest.raises(ValueError, match="softcap"):
        ab.fused_attn_bwd(do, q, k, v, o, lse, softcap=cap)
    assert torch.equal(ab.fused_attn_fwd(q, k, v, softcap=None)[0], o) and torch.equal(ab.fused_attn_fwd(q, k, v, softcap=-0.0)[0], o)


@pytest.mark.gpu
def test_a_pair_of_documents_has_two(cuda):
    """A pair that lacks one or both is refused, not taken for no documents."""
    q, k, v, do = _inputs(1, 2, 1, 4, 4, 64, BF)
    o, lse = ab.fused_attn_fwd(q, k, v)
    one = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    for docs, err in (((None, None), TypeError), ((one, None), TypeError), ((None, one), TypeError), ([None, None], TypeError),
                      ((one,), ValueError), ((one, one, one), ValueError), ((), ValueError)):
        with pytest.raises(err, match="documents"):
            ab.fused_attn_fwd(q, k, v, documents=docs)
        with pytest.raises(err, match="documents"):
            ab.fused_attn_bwd(do, q, k, v, o, lse, documents=docs)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64)])
@pytest.mark.parametrize("sq", [600, 3])
@pytest.mark.parametrize("dist", [0, 1, 3, 7, 60, 127, 200])
def test_a_bias_is_as_exact_as_its_distance(cuda, dist, sq, dtype, d):
    """Each query sees one key, some positions before it, in its own tile of keys or the one before: lse is
    that score.  Its dot product is off by up to d half steps of the sum of |q k|; slope * distance is one
    product, and the change to log2 units and back rounds both a few times (8 half steps)."""
    skv = 600
    q, k, v, _ = _inputs(1, 4, 2, sq, skv, d, dtype)
    slopes = torch.tensor([0.01, 1.0, 30.0, 1000.0], device="cuda")
    pos = torch.arange(skv, dtype=torch.int32, device="cuda")
    docs = ((pos[skv - sq:] + 5)[None].contiguous(), (pos + 5 + dist)[None].contiguous())
    o, lse = ab.fused_attn_fwd(q, k, v, causal=True, slopes=slopes, documents=docs)
    rows = torch.arange(sq, device="cuda")
    at = rows + skv - sq - dist          # the key of each row
    has = at >= 0
    assert torch.isinf(lse[:, :, ~has]).all()
    Q, K = q[0][:, has].double(), k[0].repeat_interleave(2, 0)[:, at[has]].double()
    x = (Q * K).sum(-1) / math.sqrt(d)
    bias = slopes.double()[:, None] * dist
    tol = 2.0 ** -24 * ((d + 2) * (Q * K).abs().sum(-1) / math.sqrt(d) + 8 * (x.abs() + bias))
    err = (lse[0][:, has].double() - (x - bias)).abs()
    assert (err <= tol).all(), float((err / tol).max())
    assert torch.equal(o[0, has].transpose(0, 1), v[0].repeat_interleave(2, 0)[:, at[has]])   # its weight is 1
