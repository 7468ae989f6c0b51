"""Rotary positions and attention with modified scores in 64 bits, from the formulas, with the
bounds that the kernels' 16-bit operands allow.  Test infrastructure only."""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def rope(x, pos, freq, rotary, interleaved=False, inverse=False, factor=1.0):
    """x [b, h, s, d], pos [s] or [b, s] integers, freq [rotary / 2] radians a position (float64)."""
    x = x.double().clone()
    ang = pos.to(torch.float64).reshape(-1, x.shape[2])[:, None, :, None] * freq.to(x.device)
    c, s = ang.cos() * factor, ang.sin() * factor * (-1 if inverse else 1)
    lo, hi = ((slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved
              else (slice(0, rotary // 2), slice(rotary // 2, rotary)))
    a, b = x[..., lo].clone(), x[..., hi].clone()
    x[..., lo], x[..., hi] = a * c - b * s, b * c + a * s
    return x


def seen(sq, skv, b, causal=False, prefix_lens=None, documents=None):
    """[sq, skv] truth values of batch row b."""
    i = torch.arange(sq)[:, None] + (skv - sq)
    j = torch.arange(skv)[None]
    ok = torch.ones(sq, skv, dtype=torch.bool)
    if causal:
        ok &= (j <= i) | (j < (int(prefix_lens[b]) if prefix_lens is not None else 0))
    if documents is not None:
        qd, kd = (t[b].cpu() for t in (documents if isinstance(documents, tuple) else (documents, documents)))
        ok &= (qd[:, None] == kd[None]) & (qd[:, None] >= 0)
    return ok


def attention(q, k, v, do=None, scale=None, softcap=0.0, slopes=None, causal=False, prefix_lens=None, documents=None,
              half=None, subnormal=0.0, one_tile=False):
    """Dict of o, lse (and dq, dk, dv with do) in float64 on the CPU, and for each a bound "<name>_tol"
    on the error of a computation with fp32 scores and sums whose weights p and ds are rounded to
    the inputs' type (half: half a step; subnormal: half the smallest step of the type) before
    they are multiplied, and whose results are rounded once.  one_tile: delta does not depend on the
    rounded output."""
    q, k, v = q.detach().cpu(), k.detach().cpu(), v.detach().cpu()
    half = HALF_STEP[q.dtype] if half is None else half
    if q.dtype == torch.float16:
        subnormal = 2.0 ** -25
    elif q.dtype == torch.bfloat16:
        # the exponent range of fp32: an exponential, a product or a result below its smallest normal
        # number 2^-126 may be taken as 0, so each is off by at most that much
        subnormal = 2.0 ** -126
    b, h, sq, d = q.shape
    kv, skv = k.shape[1], k.shape[2]
    grp = h // kv
    scale = 1 / math.sqrt(d) if scale is None else scale
    f32 = 2.0 ** -15   # relative error of p: scores of up to a few hundred in fp32
    out = {n: torch.zeros(b, sq, h, d, dtype=torch.float64) for n in ("o", "o_tol")}
    out["lse"] = torch.full((b, h, sq), -math.inf, dtype=torch.float64)
    out["lse_tol"] = torch.zeros(b, h, sq, dtype=torch.float64)
    for n, s, hh in (("dq", sq, h), ("dk", skv, kv), ("dv", skv, kv)):
        out[n] = torch.zeros(b, hh, s, d, dtype=torch.float64)
        out[n + "_tol"] = torch.zeros(b, hh, s, d, dtype=torch.float64)
    dist = (torch.arange(sq)[:, None] + (skv - sq) - torch.arange(skv)[None]).abs().double()
    for n in range(b):
        ok = seen(sq, skv, n, causal, prefix_lens, documents)
        qpad, kpad = ~ok.any(1), ~ok.any(0)
        for c in range(h):
            g = c // grp
            Q, K, V = q[n, c].double().clone(), k[n, g].double().clone(), v[n, g].double().clone()
            Q[qpad], K[kpad], V[kpad] = 0, 0, 0   # nothing reads them, whatever they hold
            s = Q @ K.t() * scale
            slope = torch.ones_like(s)
            size = s.abs()
            if softcap:
                t = torch.tanh(s / softcap)
                s, slope = softcap * t, 1 - t * t
                size = torch.full_like(s, softcap) + s.abs()
            if slopes is not None:
                s = s - float(slopes[c]) * dist
                size = size + float(slopes[c]) * dist
            s = s.masked_fill(~ok, -math.inf)
            m = s.amax(1, keepdim=True) if skv else s.new_full((sq, 1), -math.inf)
            lse = torch.logsumexp(s, 1) if skv else s.new_full((sq,), -math.inf)
            p = torch.where(ok, torch.exp(s - lse[:, None]), torch.zeros_like(s))
            O = p @ V
            A = p @ V.abs()
            rel = torch.clamp(size.masked_fill(~ok, 0).amax(1, keepdim=True) * 2.0 ** -22, min=f32 / 64) if skv else 0
            out["o"][n, :, c], out["lse"][n, c] = O, lse
            eo = (half + 2 * rel) * A + half * O.abs() + subnormal * V.abs().sum(0) + 2.0 ** -25 * half
            out["o_tol"][n, :, c] = eo * 1.05
            out["lse_tol"][n, c] = (2 * rel[:, 0] if skv else 0) + 2.0 ** -22 * lse.abs().nan_to_num(0, 0, 0) + 1e-6
            if do is None:
                continue
            G = do[n, :, c].detach().cpu().double().clone()
            G[qpad] = 0
            dP = G @ V.t()
            delta = (G * O).sum(1, keepdim=True)
            ddelta = (G.abs() * eo).sum(1, keepdim=True) + 2.0 ** -20 * (G.abs() * O.abs()).sum(1, keepdim=True)
            dS = p * (dP - delta) * slope
            if one_tile:
                # sum(p dp) / sum(p): what p's common error does cancels, each p's own acts on dp - delta, and
                # dp has its fp32 rounding
                ddelta = (p * (2 * rel * (dP - delta).abs() + 2.0 ** -18 * (G.abs() @ V.abs().t()))).sum(
                    1, keepdim=True)
            # ds before rounding: p and dp are fp32, delta takes the rounded output (if not one_tile)
            eS = p * slope.abs() * (ddelta + 2.0 ** -18 * (G.abs() @ V.abs().t()))
            eS = eS + (2 * rel) * (p * (dP - delta).abs()) if skv else eS
            eS = eS + half * dS.abs() + subnormal * ok
            eP = (half + 2 * rel) * p + subnormal * ok if skv else p
            out["dq"][n, c] = dS @ K * scale
            out["dq_tol"][n, c] = (eS @ K.abs() * scale) * 1.05 + half * out["dq"][n, c].abs() + subnormal
            out["dk"][n, g] += dS.t() @ Q * scale
            out["dk_tol"][n, g] += (eS.t() @ Q.abs() * scale) * 1.05
            out["dv"][n, g] += p.t() @ G
            out["dv_tol"][n, g] += (eP.t() @ G.abs()) * 1.05
    for n in ("dk", "dv"):
        out[n + "_tol"] += half * out[n].abs() + subnormal
    return out
