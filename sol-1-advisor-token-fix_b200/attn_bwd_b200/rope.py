"""Rotary positions of query and key states, forward and gradient, over ``attn_bwd_b200_rope``."""
import ctypes
import decimal
import math

import torch

from . import _lib

__all__ = ["RopeTable", "rope_table", "rope_fwd", "rope_bwd"]

_TYPES = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_FP16, torch.float32: _lib.DT_FP32}


class RopeTable:
    """Frequencies of a rotation, made once by :func:`rope_table` and kept by the caller.

    ``turns`` [rotary_dim / 2] int64 on the GPU, contiguous: each frequency as a 64-bit fixed-point
    fraction of a turn a position; ``factor`` multiplies the rotated part of a head."""

    __slots__ = ("turns", "rotary_dim", "factor")

    def __init__(self, turns, rotary_dim, factor):
        self.turns, self.rotary_dim, self.factor = turns, rotary_dim, factor


def rope_table(rotary_dim, base=10000.0, scaling=None, device="cuda"):
    """Table for angles position * f_n, f_n = base^(-2n / rotary_dim), n < rotary_dim / 2.

    ``scaling`` stretches the positions for contexts longer than the model was trained for:
      {"type": "linear", "factor": s}: every f_n divided by s;
      {"type": "base", "factor": s}: the base times s^(rotary_dim / (rotary_dim - 2)), which
        leaves the fastest pair alone and divides the slowest frequency by s;
      {"type": "ramp", "factor": s, "original_length": L, "low": a, "high": b}: pairs that turn
        fewer than a times over L positions are divided by s, pairs that turn more than b times
        are kept, linear between; both coordinates are multiplied by 0.1 ln(s) + 1 (or by
        "attention_factor" if given)."""
    if not isinstance(rotary_dim, int) or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be a positive even number, got {rotary_dim!r}")
    base = float(base)
    if not (base > 0 and math.isfinite(base)):
        raise ValueError(f"base must be positive, got {base}")
    factor, kind, s = 1.0, None, 1.0
    if scaling is not None:
        scaling = dict(scaling)
        kind = scaling.pop("type", None)
        known = {"linear": {"factor"}, "base": {"factor"},
                 "ramp": {"factor", "original_length", "low", "high", "attention_factor"}}
        if kind not in known:
            raise ValueError(f"unknown scaling type {kind!r}; known: {sorted(known)}")
        if set(scaling) - known[kind]:
            raise ValueError(f"unknown scaling keys {sorted(set(scaling) - known[kind])} for {kind!r}")
        s = float(scaling.get("factor", 0.0))
        if not (s >= 1.0 and math.isfinite(s)):
            raise ValueError(f"scaling factor must be at least 1, got {s}")
    if kind == "base" and rotary_dim == 2:
        raise ValueError("base scaling needs rotary_dim > 2")
    if kind == "ramp":
        length, low, high = (float(scaling.get(k, d)) for k, d in (("original_length", 0.0), ("low", 1.0), ("high", 32.0)))
        if not (length > 0 and high > low > -math.inf) or length == high == math.inf:
            raise ValueError("ramp scaling needs original_length > 0 and high > low")
        factor = float(scaling.get("attention_factor", 0.1 * math.log(s) + 1.0))
    # A frequency's last bits count (position * turns is exact whatever the position), and fp64 has too few:
    # 64 behind the point, through a power and a division by 2 pi, in decimal digits to spare.
    with decimal.localcontext() as ctx:
        ctx.prec = 60 + max(0, -decimal.Decimal(base).adjusted())   # base < 1: frequencies up to 1 / base
        num = decimal.Decimal
        two_pi = 2 * _pi(ctx.prec)
        exponent = num(base).ln()
        if kind == "base":
            exponent += num(s).ln() * rotary_dim / (rotary_dim - 2)
        ratio, f = (exponent * -2 / rotary_dim).exp(), [num(1)]
        for _ in range(rotary_dim // 2 - 1):
            f.append(f[-1] * ratio)
        part = 1 / num(s)
        if kind == "linear":
            f = [x * part for x in f]
        elif kind == "ramp":
            slope, start = num(length) / two_pi / (num(high) - num(low)), num(low) / (num(high) - num(low))
            keep = [min(num(1), max(num(0), x * slope - start)) for x in f]
            f = [x * (w + part * (1 - w)) for x, w in zip(f, keep)]
        unit = 2 ** 64 / two_pi
        turns = [(round(x * unit) + 2 ** 63) % 2 ** 64 - 2 ** 63 for x in f]
    return RopeTable(torch.tensor(turns, dtype=torch.int64).to(device), rotary_dim, factor)


def _pi(digits):
    """pi = 16 atan(1/5) - 4 atan(1/239) (Machin) to that many digits."""
    one = 10 ** (digits + 10)

    def atan_inverse(x):
        total, power, n = 0, one // x, 1
        while power:
            total += power // n if n % 4 == 1 else -(power // n)
            power //= x * x
            n += 2
        return total

    return decimal.Decimal(16 * atan_inverse(5) - 4 * atan_inverse(239)) / one


def _check(x, name):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(x).__name__}")
    if x.device.type != "cuda":
        raise ValueError(f"{name}: tensor must be on a CUDA device (no CPU path), got {x.device}")
    if x.dtype not in _TYPES:
        raise TypeError(f"{name}: expected bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() != 4:
        raise ValueError(f"{name}: expected [bs, heads, seq, head_dim], got {tuple(x.shape)}")


def _reaches(terms, target, budget):
    """Whether target is a sum of t * stride, lo <= t <= hi, over terms (stride, lo, hi), strides
    falling.  Layouts nest, so that each level leaves one or two t; a layout that leaves more than
    the budget of steps counts as reached."""
    if not terms:
        return target == 0
    lo = sum(s * a for s, a, _ in terms[1:])
    hi = sum(s * b for s, _, b in terms[1:])
    st, a, b = terms[0]
    for t in range(max(a, -((hi - target) // st)), min(b, (target - lo) // st) + 1):
        budget[0] -= 1
        if budget[0] < 0 or _reaches(terms[1:], target - t * st, budget):
            return True
    return False


def _extent(t):
    """Elements from a tensor's first to its last."""
    n = 1
    for size, st in zip(t.shape, t.stride()):
        n += (size - 1) * st
    return n


def _overlap(x, y):
    """Whether two tensors of one type (strides not negative) share an element's memory."""
    if x.numel() == 0 or y.numel() == 0:
        return False
    at, es = y.data_ptr() - x.data_ptr(), x.element_size()
    if at >= _extent(x) * es or -at >= _extent(y) * es:
        return False
    span = {}
    for n, st in zip(x.shape, x.stride()):
        if n > 1 and st:
            span[st] = (0, span[st][1] + n - 1) if st in span else (0, n - 1)
    for n, st in zip(y.shape, y.stride()):
        if n > 1 and st:
            a, b = span.get(st, (0, 0))
            span[st] = (a - n + 1, b)
    terms = [(st, *span[st]) for st in sorted(span, reverse=True)]
    return any(_reaches(terms, d, [4096]) for d in {at // es, -(-at // es)})


def _same_place(x, y):
    return x.data_ptr() == y.data_ptr() and all(n <= 1 or a == b for n, a, b in zip(x.shape, x.stride(), y.stride()))


def _overlaps_itself(t):
    dims, reach = sorted([(st, n) for st, n in zip(t.stride(), t.shape) if n > 1]), 0
    for st, n in dims:   # nested: every step passes what the smaller ones reach
        if st <= reach:
            break
        reach += (n - 1) * st
    else:
        return False
    if t.numel() == 0:
        return False
    if dims[0][0] == 0:
        return True
    dims.reverse()
    budget = [4096]
    for i, (st, n) in enumerate(dims):   # two elements whose first different index is this one
        rest = [(s, 1 - m, m - 1) for s, m in dims[i + 1:]]
        reach = sum(s * b for s, _, b in rest)
        if any(_reaches(rest, d * st, budget) for d in range(1, min(n - 1, reach // st) + 1)):
            return True
    return False


def _check_places(ins, outs, given):
    """Refuses results that the caller gave (the names in given) where they overlap an input, other than
    their own in its own place, or each other."""
    names = ("query", "key")
    own = [o is not None and n in given and _same_place(o, x) for x, o, n in zip(ins, outs, names)]
    for i, name in enumerate(names):
        if name not in given:
            continue
        for j, x in enumerate(ins):
            # (an input that is its own result is looked at as that, below)
            if x is not None and not own[j] and _overlap(outs[i], x):
                raise ValueError(f"out: {name} overlaps the input {names[j]}" + (" in another order" if i == j else ""))
    if len(given) == 2 and _overlap(*outs):
        raise ValueError("out: query and key overlap")


def _rotate(q, k, position_ids, table, interleaved, inverse, out):
    if isinstance(table, RopeTable):
        args = (q, k, position_ids, table.turns, table.rotary_dim, table.factor, bool(interleaved), inverse)
        if out is None:
            r = _lib.bound("rope", *args)
        else:
            r = _lib.bound("rope_into", *args, *out) if isinstance(out, (tuple, list)) and len(out) == 2 else None
        if r is not None:
            return r
    if not isinstance(table, RopeTable):
        raise TypeError(f"table: expected a RopeTable (rope_table(...)), got {type(table).__name__}")
    turns = table.turns
    if not isinstance(turns, torch.Tensor) or turns.dtype != torch.int64:
        raise TypeError("table: turns must be an int64 tensor")
    if not isinstance(table.rotary_dim, int) or tuple(turns.shape) != (table.rotary_dim // 2,) or table.rotary_dim % 2:
        raise ValueError(f"table: turns of {tuple(turns.shape)} do not belong to {table.rotary_dim} rotated elements")
    if not turns.is_contiguous():
        raise ValueError("table: turns must be contiguous")
    names = ("query", "key")
    xs = [x for x in (q, k) if x is not None]
    if not xs:
        raise ValueError("nothing to rotate: both tensors are None")
    for x, name in zip((q, k), names):
        if x is not None:
            _check(x, name)
    first = xs[0]
    bs, _, seq, d = first.shape
    for x in xs:
        if (x.shape[0], x.shape[2], x.shape[3]) != (bs, seq, d) or x.dtype != first.dtype or x.device != first.device:
            raise ValueError("query and key must agree in batch, positions, head_dim, dtype and device, got "
                             f"{[(tuple(x.shape), x.dtype, x.device) for x in xs]}")
    if table.rotary_dim > d:
        raise ValueError(f"table rotates {table.rotary_dim} elements, heads have {d}")
    if turns.device != first.device:
        raise ValueError(f"table is on {turns.device}, tensors on {first.device}")
    if not isinstance(position_ids, torch.Tensor) or position_ids.dtype not in (torch.int64, torch.int32):
        raise TypeError("position_ids: expected an int64 or int32 tensor")
    if position_ids.device != first.device:
        raise ValueError(f"position_ids is on {position_ids.device}, tensors on {first.device}")
    shape = tuple(position_ids.shape)
    if shape not in ((seq,), (1, seq), (bs, seq)):
        raise ValueError(f"position_ids: expected [{seq}], [1, {seq}] or [{bs}, {seq}], got {shape}")
    with torch.cuda.device(first.device):
        pos = position_ids.to(torch.int64).contiguous()
        per_batch = pos.dim() == 2 and pos.shape[0] == bs and bs > 1
        outs, given = [], []
        if out is None:
            out = (None, None)
        elif not isinstance(out, (tuple, list)) or len(out) != 2:
            raise ValueError("out: expected a pair (query, key) of tensors or None")
        ins = []
        for x, o, name in zip((q, k), out, names):
            if x is None:
                if o is not None:
                    raise ValueError(f"out: {name} was not given")
                ins.append(None)
                outs.append(None)
                continue
            if x.stride(3) != 1 and d > 1:
                x = x.contiguous()
            if o is None:
                o = torch.empty_like(x)   # same order in memory as the input
                if o.stride(3) != 1:
                    o = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            else:
                if (not isinstance(o, torch.Tensor) or o.shape != x.shape or o.dtype != x.dtype or
                        o.device != x.device or (o.stride(3) != 1 and d > 1)):
                    raise ValueError(f"out: {name} must match the input's shape, dtype and device, head elements contiguous")
                if _overlaps_itself(o):
                    raise ValueError(f"out: {name} overlaps itself")
                given.append(name)
            ins.append(x)
            outs.append(o)
        _check_places(ins, outs, given)
        a = _lib.RopeArgs()
        a.bs, a.seq, a.head_dim, a.rotary_dim = bs, seq, d, table.rotary_dim
        a.q_heads = q.shape[1] if q is not None else 0
        a.k_heads = k.shape[1] if k is not None else 0
        a.dtype = _TYPES[first.dtype]
        a.interleaved, a.inverse = int(bool(interleaved)), int(inverse)
        a.factor = table.factor
        a.position_stride = seq if per_batch else 0
        for t, dst in zip((ins[0], ins[1], outs[0], outs[1]), (a.q_in, a.k_in, a.q_out, a.k_out)):
            if t is not None:
                dst[:] = t.stride()[:3]
        ptr = [0 if t is None else t.data_ptr() for t in (ins[0], ins[1])]
        optr = [0 if t is None else t.data_ptr() for t in outs]
        _lib.call("attn_bwd_b200_rope", ctypes.byref(a), ptr[0], ptr[1], pos.data_ptr(), turns.data_ptr(),
                  optr[0], optr[1], torch.cuda.current_stream().cuda_stream)
    return outs[0], outs[1]


def rope_fwd(query_states, key_states, position_ids, table, interleaved=False, out=None):
    """Rotates query_states [bs, heads, seq, d] and key_states [bs, kv_heads, seq, d] (either may
    be None) at position_ids ([seq], [1, seq] or [bs, seq]; any integer, and the angle of position p is
    off by |p| * 2^-65 + 2^-33 turns at most besides fp32's own rounding) in one launch.  Heads of at most 4096.

    The first ``table.rotary_dim`` elements of a head are rotated, the rest is copied.  Pairs are
    (n, n + rotary_dim / 2), or neighbours with ``interleaved``.  bfloat16, float16 or float32;
    any strides (heads inside positions or positions inside heads); the results keep the inputs' order in
    memory.  ``out`` takes preallocated results and may be the inputs themselves; results that
    otherwise overlap an input, each other or themselves are refused."""
    return _rotate(query_states, key_states, position_ids, table, interleaved, False, out)


def rope_bwd(grad_query, grad_key, position_ids, table, interleaved=False, out=None):
    """Gradients of :func:`rope_fwd`'s inputs from those of its results: the inverse rotation,
    times the table's factor.  Arguments as there."""
    return _rotate(grad_query, grad_key, position_ids, table, interleaved, True, out)
