"""What is measured of the operators around the attention backward: rotary positions and fused attention.

A training step of a GQA layer rotates its queries and keys, attends, and on the way back takes
the gradients through both.  The cases here are those passes: ``rope_fwd`` / ``rope_bwd`` (one
rotation of queries and keys, or of their gradients), ``attn_fwd`` (one forward call: prompts,
chunks of new tokens and single tokens over a long cache) and ``attn_train`` (forward and
backward of one layer, as a training step calls them).  Scores may be capped by a tanh, get a
bias that falls with distance, and be masked causally, by documents or by a prefix.

``run`` computes a case in plain torch operations, or, where ``own`` is true, by the calls of the
``attn_bwd_b200`` package.  ``exact`` is the definition in 64 bits.
"""
import math
import os
import random
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def _rope(name, op, bs, s, heads, kv, dim, rotary, dtype, interleaved=False, scaling="none", start=0, layout="bshd"):
    return {"name": name, "op": op, "bs": bs, "sq": s, "heads": heads, "kv_heads": kv, "dim": dim, "rotary": rotary,
            "dtype": dtype, "interleaved": interleaved, "scaling": scaling, "start": start, "layout": layout}


def _attn(name, op, bs, sq, skv, heads, kv, dim, dtype, causal=False, softcap=0.0, slopes=False, prefix=False,
          docs=0, layout="bshd"):
    return {"name": name, "op": op, "bs": bs, "sq": sq, "skv": skv, "heads": heads, "kv_heads": kv, "dim": dim,
            "dtype": dtype, "causal": causal, "softcap": softcap, "slopes": slopes, "prefix": prefix, "docs": docs,
            "layout": layout}


def listed():
    return [
        # one new token for each of 8 sequences of a served layer, far into their contexts
        _rope("rope_tokens", "rope_fwd", 8, 1, 80, 8, 128, 128, "bf16", start=30011),
        # the layer's ragged training batch, half of each head rotated, neighbouring pairs
        _rope("rope_ragged_part", "rope_fwd", 12, 467, 80, 8, 128, 64, "fp16", interleaved=True, layout="bhsd"),
        # two long documents whose positions pass the length that the frequencies were made for
        _rope("rope_long_scaled", "rope_fwd", 2, 16001, 80, 8, 128, 128, "bf16", scaling="ramp", start=100003),
        # the gradients of the layer's largest training batch on their way back through the rotation
        _rope("rope_grad", "rope_bwd", 48, 640, 80, 8, 128, 128, "bf16"),
        # one new token for each of 4 sequences over a cache of 8191: reads the cache once
        _attn("attn_token", "attn_fwd", 4, 1, 8191, 80, 8, 128, "bf16", causal=True, layout="bhsd"),
        # a short chunk of new tokens behind one long context, capped scores
        _attn("attn_chunk", "attn_fwd", 1, 77, 32013, 40, 8, 128, "fp16", causal=True, softcap=30.0),
        # a prompt
        _attn("attn_prompt", "attn_fwd", 1, 4096, 4096, 80, 8, 128, "bf16", causal=True),
        # packed documents with a padded end, a bias that falls with distance, small heads
        _attn("attn_packed_bias", "attn_fwd", 2, 5003, 5003, 32, 8, 64, "bf16", causal=True, slopes=True, docs=900),
        # the smallest training batch
        _attn("train_small", "attn_train", 2, 64, 96, 80, 8, 128, "bf16"),
        # ragged training batch, queries fewer than keys, a prefix that all queries see
        _attn("train_ragged_prefix", "attn_train", 12, 301, 467, 80, 8, 128, "bf16", causal=True, slopes=True,
              prefix=True),
        # the largest training batch, capped scores
        _attn("train_capped", "attn_train", 48, 640, 640, 80, 8, 128, "bf16", causal=True, softcap=40.0),
        # one long packed row of documents
        _attn("train_packed", "attn_train", 1, 8192, 8192, 80, 8, 128, "bf16", causal=True, docs=2500),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope_fwd", "rope_bwd", "attn_fwd", "attn_fwd", "attn_train", "attn_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    kv = rng.choice([1, 2, 3, 4, 8, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 8, 10])
    layout = rng.choice(["bshd", "bhsd"])
    if op.startswith("rope"):
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        tokens = _log(rng, 1, 32000)
        bs = min(tokens, rng.choice([1, 2, 3, 7, 16]))
        c = _rope("", op, bs, max(1, tokens // bs), heads, kv, dim, dim if rng.random() < 0.6 else dim // 2,
                  rng.choice([dtype, dtype, "fp32"]), rng.random() < 0.5,
                  rng.choice(["none", "linear", "base", "ramp"]), _log(rng, 1, 1000000) - 1, layout)
        while c["bs"] * c["sq"] * (heads + kv) * dim > 345_000_000:
            c["sq"] = max(1, c["sq"] // 2)
    else:
        dim = rng.choice([64, 128, 128])
        docs = 0
        causal = rng.random() < 0.7
        softcap = rng.choice([0.0, 0.0, 15.0, 30.0, 50.0])
        slopes = rng.random() < 0.3
        bs = rng.choice([1, 1, 2, 3, 5, 8, 16])
        if op == "attn_fwd" and rng.random() < 0.5:      # serving: few new tokens over a cache
            sq = rng.choice([1, 1, 1, 2, 5, 16, _log(rng, 2, 300)])
            skv = sq + _log(rng, 1, 40000)
            limit = 1.5e11
        else:
            sq = _log(rng, 1 if op == "attn_fwd" else 8, 6000)
            skv = sq if rng.random() < 0.6 else sq + _log(rng, 1, 2000)
            docs = rng.choice([0, 0, max(2, sq // rng.choice([1, 2, 4, 9]))])
            limit = 1.2e12
        prefix = causal and rng.random() < 0.3
        while 14.0 * bs * heads * sq * skv * dim > limit and (bs > 1 or heads > kv or sq > 64):
            if bs > 1:
                bs = bs // 2
            elif heads > kv:
                heads = max(kv, heads // 2 // kv * kv)
            else:
                skv, sq = skv - sq // 2, sq - sq // 2
        c = _attn("", op, bs, sq, skv, heads, kv, dim, dtype, causal, softcap, slopes, prefix, docs, layout)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def _documents(case):
    """Document number of each key, [bs, skv] as lists: documents of random lengths about
    case["docs"], and -1 (no document) behind the last one of a row: up to a twentieth of it."""
    r = random.Random(case["skv"] * 1009 + case["docs"])
    rows = []
    for _ in range(case["bs"]):
        n = case["skv"] - r.randint(0, case["skv"] // 20)
        row = []
        while len(row) < n:
            d = len(row) and row[-1] + 1
            row += [d] * min(n - len(row), max(1, int(case["docs"] * r.uniform(0.3, 1.7))))
        rows.append(row + [-1] * (case["skv"] - n))
    return rows


def _prefixes(case):
    r = random.Random(case["skv"] * 31 + case["bs"])
    return [r.randint(0, case["skv"] // 2) for _ in range(case["bs"])]


def _tensor(g, b, s, h, d, dtype, layout, std=1.0):
    """[b, h, s, d], stored with heads inside tokens ("bshd") or tokens inside heads ("bhsd")."""
    shape = (b, s, h, d) if layout == "bshd" else (b, h, s, d)
    t = torch.randn(shape, device="cuda", generator=g).mul_(std).to(dtype)
    return t.transpose(1, 2) if layout == "bshd" else t


_SCALING = {"none": None, "linear": {"type": "linear", "factor": 4.0}, "base": {"type": "base", "factor": 8.0},
            "ramp": {"type": "ramp", "factor": 8.0, "original_length": 8192, "low": 1.0, "high": 32.0}}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, lay = _DT[case["dtype"]], case["layout"]
    b, sq, h, kv, d = case["bs"], case["sq"], case["heads"], case["kv_heads"], case["dim"]
    if case["op"].startswith("rope"):
        st = {"case": case, "q": _tensor(g, b, sq, h, d, dt, lay), "k": _tensor(g, b, sq, kv, d, dt, lay),
              "pos": (torch.arange(sq, device="cuda") + case["start"])[None]
              + torch.randint(0, 97, (b, 1), device="cuda", generator=g)}
        if own:
            ab = _package()
            st["table"] = ab.rope_table(case["rotary"], base=10000.0, scaling=_SCALING[case["scaling"]], device="cuda")
        else:
            st["freq"], st["factor"] = _frequencies(case)
        return st
    skv = case["skv"]
    # capped layers meet larger scores
    st = {"case": case, "q": _tensor(g, b, sq, h, d, dt, lay, 3.0 if case["softcap"] else 1.0),
          "k": _tensor(g, b, skv, kv, d, dt, lay), "v": _tensor(g, b, skv, kv, d, dt, lay)}
    mods = {"scale": 1.0 / math.sqrt(d), "softcap": case["softcap"], "causal": case["causal"]}
    mods["slopes"] = (torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda")
                      if case["slopes"] else None)
    mods["prefix_lens"] = (torch.tensor(_prefixes(case), dtype=torch.int32, device="cuda")
                           if case["prefix"] else None)
    mods["documents"] = None
    if case["docs"]:
        kd = torch.tensor(_documents(case), dtype=torch.int32, device="cuda")
        mods["documents"] = (kd[:, skv - sq:].contiguous(), kd)
    st["mods"] = mods
    if case["op"] == "attn_train":
        st["do"] = torch.randn(b, sq, h, d, device="cuda", generator=g).to(dt)
    return st


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sol-1-advisor-token-fix_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import attn_bwd_b200
    return attn_bwd_b200


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    if "pos" in state:
        return _plain_rope(state)
    return _plain_attention(state)


def _run_own(st):
    ab = _package()
    case = st["case"]
    if case["op"] == "rope_fwd":
        return ab.rope_fwd(st["q"], st["k"], st["pos"], st["table"], interleaved=case["interleaved"])
    if case["op"] == "rope_bwd":
        return ab.rope_bwd(st["q"], st["k"], st["pos"], st["table"], interleaved=case["interleaved"])
    o, lse = ab.fused_attn_fwd(st["q"], st["k"], st["v"], **st["mods"])
    if case["op"] == "attn_fwd":
        return o, lse
    dq, dk, dv = ab.fused_attn_bwd(st["do"], st["q"], st["k"], st["v"], o, lse, **st["mods"])
    return o, lse, dq, dk, dv


# ------------------------------------------------------------------ the plain forms
def _frequencies(case):
    """Angles a position (float64) and the factor on both coordinates."""
    n = case["rotary"]
    sc = _SCALING[case["scaling"]]
    base = 10000.0
    if sc and sc["type"] == "base":
        base *= sc["factor"] ** (n / (n - 2.0))
    f = base ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
    factor = 1.0
    if sc and sc["type"] == "linear":
        f = f / sc["factor"]
    if sc and sc["type"] == "ramp":
        turns = sc["original_length"] * f / (2 * math.pi)
        keep = ((turns - sc["low"]) / (sc["high"] - sc["low"])).clamp(0, 1)
        f = f * keep + f / sc["factor"] * (1 - keep)
        factor = 0.1 * math.log(sc["factor"]) + 1.0
    return f.cuda(), factor


def _turn(x, cos, sin, case):
    """x [b, h, s, d] rotated by angles of [b, 1, s, rotary / 2]."""
    n, y = case["rotary"], x.clone()
    if case["interleaved"]:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        y[..., 0:n:2], y[..., 1:n:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :n // 2], x[..., n // 2:n]
        y[..., :n // 2], y[..., n // 2:n] = a * cos - b * sin, b * cos + a * sin
    return y


def _plain_rope(st):
    case = st["case"]
    angle = st["pos"].double()[:, None, :, None] * st["freq"]
    cos, sin = (angle.cos() * st["factor"]).float(), (angle.sin() * st["factor"]).float()
    if case["op"] == "rope_bwd":
        sin = -sin
    return tuple(_turn(st[n].float(), cos, sin, case).to(st[n].dtype) for n in ("q", "k"))


def _allowed(case, mods, b):
    """[sq, skv] truth values of one batch row, or None where every query sees every key."""
    sq, skv = case["sq"], case["skv"]
    ok = None
    if case["causal"]:
        i = torch.arange(sq, device="cuda")[:, None] + (skv - sq)
        j = torch.arange(skv, device="cuda")[None]
        ok = j <= i
        if mods["prefix_lens"] is not None:
            ok = ok | (j < mods["prefix_lens"][b])
    if mods["documents"] is not None:
        qd, kd = mods["documents"][0][b][:, None], mods["documents"][1][b][None]
        same = (qd == kd) & (qd >= 0)
        ok = same if ok is None else ok & same
    return ok


def _plain_attention(st):
    case, mods = st["case"], st["mods"]
    sq, skv, h, kv = case["sq"], case["skv"], case["heads"], case["kv_heads"]
    grp, cap = h // kv, case["softcap"]
    rows = {n: [] for n in ("o", "lse", "dq", "dk", "dv")}
    for b in range(case["bs"]):
        q = st["q"][b].float().reshape(kv, grp * sq, -1)              # the heads of a group share k and v
        k, v = st["k"][b].float(), st["v"][b].float()
        x = torch.matmul(q, k.transpose(1, 2)).mul_(mods["scale"])
        t = None
        if cap:
            t = torch.tanh(x.div_(cap))
            x = t * cap
        x = x.view(h, sq, skv)
        if mods["slopes"] is not None:
            dist = (torch.arange(sq, device="cuda")[:, None] + (skv - sq) - torch.arange(skv, device="cuda")).abs()
            x = x - mods["slopes"][:, None, None] * dist
        ok = _allowed(case, mods, b)
        if ok is not None:
            x = x.masked_fill_(~ok, -math.inf)
        m = x.amax(-1, keepdim=True)
        p = torch.exp(x.sub_(torch.where(m == -math.inf, 0.0, m)))
        l = p.sum(-1, keepdim=True)
        p = p.div_(torch.where(l == 0, 1.0, l)).view(kv, grp * sq, skv)
        del x
        o = torch.matmul(p, v)
        rows["o"].append(o.view(h, sq, -1).transpose(0, 1).to(st["q"].dtype))
        rows["lse"].append((m + torch.log(l)).view(h, sq))
        if case["op"] == "attn_train":
            do = st["do"][b].float().transpose(0, 1).reshape(kv, grp * sq, -1)
            rows["dv"].append(torch.matmul(p.transpose(1, 2), do).to(st["v"].dtype))
            ds = torch.matmul(do, v.transpose(1, 2)).sub_((o * do).sum(-1, keepdim=True)).mul_(p)
            if cap:
                ds = ds.mul_(1 - t * t)
            rows["dq"].append(torch.matmul(ds, k).mul_(mods["scale"]).view(h, sq, -1).to(st["q"].dtype))
            rows["dk"].append(torch.matmul(ds.transpose(1, 2), q).mul_(mods["scale"]).to(st["k"].dtype))
    names = ("o", "lse") if case["op"] == "attn_fwd" else ("o", "lse", "dq", "dk", "dv")
    return tuple(torch.stack(rows[n]) for n in names)


# ------------------------------------------------------------------ what a pass cannot do without
def _pairs(case):
    """Pairs of a query and a key that it sees, over the batch (one head)."""
    sq, skv, n = case["sq"], case["skv"], 0
    docs = _documents(case) if case["docs"] else None
    pre = _prefixes(case) if case["prefix"] else [0] * case["bs"]
    for b in range(case["bs"]):
        if docs is None and not case["causal"]:
            n += sq * skv
        elif docs is None:
            n += sum(max(min(skv, i + skv - sq + 1), pre[b]) for i in range(sq))
        else:
            first = {}
            for j, d in enumerate(docs[b]):
                first.setdefault(d, j)
            last = {d: j for j, d in enumerate(docs[b])}
            for i in range(skv - sq, skv):
                d = docs[b][i]
                if d >= 0:
                    hi = last[d] + 1
                    if case["causal"]:
                        hi = min(hi, max(i + 1, pre[b]))
                    n += max(0, hi - first[d])
    return n


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    b, sq, h, kv, d = case["bs"], case["sq"], case["heads"], case["kv_heads"], case["dim"]
    if case["op"].startswith("rope"):
        n = b * sq * (h + kv)
        return {"bytes": 2 * n * d * es + 8 * b * sq, "flops": 3 * n * case["rotary"]}
    skv = case["skv"]
    q, k = b * sq * h * d * es, b * skv * kv * d * es
    extra = (b * (sq + skv) * 4 if case["docs"] else 0) + (h * 4 if case["slopes"] else 0)
    mm = 2 * h * d * _pairs(case)
    if case["op"] == "attn_fwd":
        return {"bytes": 2 * q + 2 * k + b * h * sq * 4 + extra, "flops": 2 * mm}
    # reads q, k, v and the output's gradient, writes the output, its row statistics and three gradients
    return {"bytes": 4 * q + 4 * k + b * h * sq * 4 + extra, "flops": 7 * mm}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    global own
    if case["op"].startswith("attn") and case["bs"] * case["heads"] * case["sq"] * case["skv"] > 6_000_000_000:
        return None
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if case["op"].startswith("rope"):
        ang = torch.einsum("bs,f->bsf", st["pos"].to(torch.float64), st["freq"])
        z = torch.polar(torch.full_like(ang, st["factor"]), -ang if case["op"] == "rope_bwd" else ang)[:, None]
        out = []
        for x in (st["q"], st["k"]):
            x = x.to(torch.float64)
            n = case["rotary"]
            rot = x[..., :n]
            pair = rot.unflatten(-1, (n // 2, 2)) if case["interleaved"] else rot.unflatten(-1, (2, n // 2)).transpose(-1, -2)
            w = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
            w = w if case["interleaved"] else w.transpose(-1, -2)
            out.append(torch.cat([w.flatten(-2), x[..., n:]], -1))
        return tuple(out)
    mods = st["mods"]
    b, sq, skv, h, kv, d = (case[n] for n in ("bs", "sq", "skv", "heads", "kv_heads", "dim"))
    train = case["op"] == "attn_train"
    f64 = dict(dtype=torch.float64, device="cuda")
    o, lse = torch.zeros(b, sq, h, d, **f64), torch.zeros(b, h, sq, **f64)
    dq, dk, dv = torch.zeros(b, h, sq, d, **f64), torch.zeros(b, kv, skv, d, **f64), torch.zeros(b, kv, skv, d, **f64)
    i, j = torch.arange(sq, device="cuda").view(-1, 1) + (skv - sq), torch.arange(skv, device="cuda").view(1, -1)
    for n in range(b):
        see = torch.ones(sq, skv, dtype=torch.bool, device="cuda")
        if case["causal"]:
            see &= j < torch.clamp(i + 1, min=int(mods["prefix_lens"][n]) if case["prefix"] else 0)
        if case["docs"]:
            qd, kd = (t[n] for t in mods["documents"])
            see &= (qd.view(-1, 1) == kd.view(1, -1)) & (qd.view(-1, 1) != -1)
        for c in range(h):
            g = c // (h // kv)
            Q, K, V = st["q"][n, c].double(), st["k"][n, g].double(), st["v"][n, g].double()
            s = Q @ K.t() * mods["scale"]
            slope = None
            if case["softcap"]:
                th = torch.tanh(s / case["softcap"])
                s, slope = case["softcap"] * th, 1 - th * th
            if case["slopes"]:
                s = s - mods["slopes"][c].double() * (i - j).abs()
            s = torch.where(see, s, torch.full_like(s, -math.inf))
            lse[n, c] = torch.logsumexp(s, -1)
            P = torch.where(see, torch.exp(s - lse[n, c].view(-1, 1)), torch.zeros_like(s))
            O = P @ V
            o[n, :, c] = O
            if train:
                G = st["do"][n, :, c].double()
                dv[n, g] += P.t() @ G
                dP = G @ V.t()
                S = P * (dP - (P * dP).sum(-1, keepdim=True))
                if slope is not None:
                    S = S * slope
                dq[n, c] = S @ K * mods["scale"]
                dk[n, g] += S.t() @ Q * mods["scale"]
    return (o, lse, dq, dk, dv) if train else (o, lse)
