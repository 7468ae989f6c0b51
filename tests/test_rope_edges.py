"""Rotary positions: tables and results that a caller makes itself."""
import decimal
import math

import pytest
import torch

import attn_bwd_b200 as ab

BF = torch.bfloat16


def _tables(dev):
    """(table, error): turns that do not belong to the elements that are to be rotated."""
    t = torch.arange(64, dtype=torch.int64, device=dev)
    return [(ab.RopeTable(t[:31], 64, 1.0), ValueError), (ab.RopeTable(t[:33], 64, 1.0), ValueError),
            (ab.RopeTable(t[:0], 64, 1.0), ValueError), (ab.RopeTable(t[:32][None], 64, 1.0), ValueError),
            (ab.RopeTable(t[::2], 64, 1.0), ValueError), (ab.RopeTable(t[:31], 63, 1.0), ValueError),
            (ab.RopeTable(t[:32], 64.0, 1.0), ValueError), (ab.RopeTable(t[:32].double(), 64, 1.0), TypeError),
            (ab.RopeTable(t[:32].int(), 64, 1.0), TypeError), (ab.RopeTable([0] * 32, 64, 1.0), TypeError)]


def test_table_of_another_size_is_refused():
    """Before anything else is looked at (a short table would be read behind its end)."""
    x = torch.zeros(1, 2, 3, 64)
    for table, err in _tables("cpu"):
        for fn in (ab.rope_fwd, ab.rope_bwd):
            with pytest.raises(err, match="turns"):
                fn(x, x, torch.arange(3), table)


@pytest.mark.gpu
def test_table_of_another_size_is_refused_on_the_gpu(cuda):
    x = torch.zeros(1, 2, 3, 64, dtype=BF, device="cuda")
    pos = torch.arange(3, device="cuda")
    for table, err in _tables("cuda"):
        for args in ((x, x), (x, None), (None, x)):
            with pytest.raises(err, match="turns"):
                ab.rope_fwd(*args, pos, table)
            with pytest.raises(err, match="turns"):
                ab.rope_fwd(*args, pos, table, out=tuple(None if a is None else torch.empty_like(a) for a in args))
    ok = ab.RopeTable(torch.arange(32, dtype=torch.int64, device="cuda"), 64, 1.0)
    assert ab.rope_fwd(x, x, pos, ok)[0].shape == x.shape


# ------------------------------------------------------------------ results that overlap
def _cells(t):
    """Addresses of a small tensor's elements, in bytes."""
    idx = torch.zeros(t.shape, dtype=torch.int64)
    for n, (size, st) in enumerate(zip(t.shape, t.stride())):
        shape = [1] * t.dim()
        shape[n] = size
        idx = idx + (torch.arange(size) * st * t.element_size()).reshape(shape)
    return t.data_ptr() + idx.flatten()


def test_overlap_against_every_address():
    """Random small layouts in one buffer: what the check says is what their addresses say."""
    g = torch.Generator().manual_seed(0)
    buf = torch.zeros(4096, dtype=BF)
    rnd = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))
    met = own = 0
    for _ in range(3000):
        ts = []
        for _ in range(2):
            shape = [rnd(1, 4) for _ in range(4)]
            if rnd(0, 2):   # nested, as layouts are, in any order and with gaps
                stride, st = [0] * 4, 1
                for n in torch.randperm(4, generator=g).tolist():
                    stride[n] = st
                    st *= shape[n] + rnd(0, 2)
            else:
                stride = [rnd(0, 12) for _ in range(4)]
            ts.append(buf.as_strided(shape, stride, rnd(0, 60)))
        a, b = (set(_cells(t).tolist()) for t in ts)
        assert ab.rope._overlap(*ts) == bool(a & b), [(t.shape, t.stride(), t.storage_offset()) for t in ts]
        met += bool(a & b)
        for t, cells in zip(ts, (a, b)):
            assert ab.rope._overlaps_itself(t) == (len(cells) < t.numel()), (t.shape, t.stride())
            own += len(cells) < t.numel()
    assert 500 < met < 2800 and own > 500
    big = torch.empty(2, 88, 16001, 128, dtype=BF, device="meta")   # sizes of a real layer: no search
    assert not ab.rope._overlaps_itself(big) and not ab.rope._overlaps_itself(big.transpose(1, 2))


@pytest.mark.gpu
def test_overlapping_results(cuda):
    g = torch.Generator().manual_seed(1)
    fused = torch.randn(2, 9, 8, 64, generator=g).to(BF).cuda()   # [bs, seq, 4 + 2 + 2 heads, d]
    q, k = fused[:, :, :4].transpose(1, 2), fused[:, :, 4:6].transpose(1, 2)
    pos, t = torch.arange(9, device="cuda"), ab.rope_table(64)
    want = ab.rope_fwd(q, k, pos, t)
    rest = fused[:, :, 6:].clone()
    out = ab.rope_fwd(q, k, pos, t, out=(q, k))                    # in place in one buffer: nothing overlaps
    assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(fused[:, :, 6:], rest)
    x = torch.randn(1, 2, 20, 64, generator=g).to(BF).cuda()
    a, b, c = x[:, :, :9], x[:, :, 1:10], x[:, :, 10:19]
    for bad in (dict(q=a, k=None, out=(b, None)),                  # its own input, a position on
                dict(q=a, k=c, out=(c, torch.empty_like(c))),      # the other input
                dict(q=a, k=c, out=(torch.empty_like(a), b)),
                dict(q=a.clone(), k=c.clone(), out=(a, b)),        # each other
                dict(q=a.clone(), k=c.clone(), out=(a, a)),
                dict(q=a.clone(), k=None, out=(x.as_strided((1, 2, 9, 64), (0, 64, 64, 1)), None)),
                dict(q=a, k=None, out=(x.as_strided((1, 2, 9, 64), (64, 64, 128, 1)), None))):
        with pytest.raises(ValueError, match="overlap"):
            ab.rope_fwd(bad["q"], bad["k"], pos, t, out=bad["out"])
    got = ab.rope_fwd(a, None, pos, t, out=(c, None))[0]           # beside the input in its buffer
    assert torch.equal(got, ab.rope_fwd(a, None, pos, t)[0])


# ------------------------------------------------------------------ the last bits of a frequency
PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798")


def _bracketed(turns, equation):
    """Whether a rising function of the frequency (radians a position, 90 digits) passes 1 within one unit
    of 2^-64 turns."""
    with decimal.localcontext() as ctx:
        ctx.prec, ctx.Emax, ctx.Emin = 95, decimal.MAX_EMAX, decimal.MIN_EMIN
        at = lambda n: equation(decimal.Decimal(n) / 2 ** 64 * 2 * PI)
        return at(turns - 1) < 1 < at(turns + 1)


@pytest.mark.parametrize("rotary,base", [(128, 10000.0), (64, 500000.0), (80, 10000.0), (10, 123.456), (256, 1e8), (2, 7.0), (4096, 10000.0)])
def test_turns_to_the_last_bit(rotary, base):
    """f = base^(-2n / rotary) is the solution of f^rotary base^2n = 1: whole powers only."""
    b, s = decimal.Decimal(base), decimal.Decimal("3.5")
    steps = range(0, rotary // 2, max(1, rotary // 128))
    plain = ab.rope_table(rotary, base=base, device="cpu").turns.tolist()
    linear = ab.rope_table(rotary, base=base, scaling={"type": "linear", "factor": 3.5}, device="cpu").turns.tolist()
    for n in steps:
        assert _bracketed(plain[n], lambda f: f ** rotary * b ** (2 * n)), n
        assert _bracketed(linear[n], lambda f: (f * s) ** rotary * b ** (2 * n)), n
    if rotary > 2:
        # (base s^(r / (r - 2)))^(-2n / r): f^(r (r - 2)) base^(2n (r - 2)) s^(2n r) = 1
        scaled = ab.rope_table(rotary, base=base, scaling={"type": "base", "factor": 3.5}, device="cpu").turns.tolist()
        for n in steps:
            assert _bracketed(scaled[n], lambda f: f ** (rotary * (rotary - 2)) * b ** (2 * n * (rotary - 2)) * s ** (2 * n * rotary)), n


def test_ramp_turns_to_the_last_bit():
    plain = ab.rope_table(128, device="cpu").turns.tolist()
    ramp = ab.rope_table(128, scaling={"type": "ramp", "factor": 8.0, "original_length": 4096}, device="cpu").turns.tolist()
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        for n, (a, b) in enumerate(zip(plain, ramp)):
            # f^128 10000^2n = 1 solved from the fp64 value by Newton's method
            f = decimal.Decimal(10000.0 ** (-2 * n / 128))
            for _ in range(3):
                f -= f * (f ** 128 * decimal.Decimal(10000) ** (2 * n) - 1) / 128
            w = min(decimal.Decimal(1), max(decimal.Decimal(0), (4096 * f / (2 * PI) - 1) / 31))
            want = (f * w + f / 8 * (1 - w)) / (2 * PI) * 2 ** 64
            assert abs(want - b) <= 1, n
            assert abs(f / (2 * PI) * 2 ** 64 - a) <= 1, n


def test_tables_of_other_bases():
    one = ab.rope_table(8, base=1.0, device="cpu").turns.tolist()
    assert len(set(one)) == 1 and abs(one[0] / 2 ** 64 - 1 / (2 * math.pi)) < 1e-15
    low = ab.rope_table(8, base=1e-4, device="cpu").turns.tolist()   # frequencies above a turn a position: what is behind the point
    for t, f in zip(low, (1, 10, 100, 1000)):
        assert abs((t % 2 ** 64) / 2 ** 64 - math.fmod(f / (2 * math.pi), 1.0)) < 1e-12
    with pytest.raises(ValueError, match="ramp"):
        ab.rope_table(8, scaling={"type": "ramp", "factor": 2.0, "original_length": 10, "low": -math.inf}, device="cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("start", [10 ** 9, 10 ** 12, -10 ** 12 + 7, 2 ** 40 + 12345])
def test_far_positions_to_the_last_bit(cuda, start):
    """Angles of far positions from frequencies of 60 digits.  The table's half unit costs |position| / 2 *
    2^-64 turns, the angle's own 32 bits 2^-33 of one, fp32 half a step each of angle, sine and product."""
    d, s = 128, 9
    x = torch.randn(1, 2, s, d, generator=torch.Generator().manual_seed(2)).cuda()
    pos = torch.arange(s, device="cuda") + start
    got, _ = ab.rope_fwd(x, None, pos, ab.rope_table(d))
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        ln = decimal.Decimal(10000).ln()
        f = [(ln * (-2 * n) / d).exp() / (2 * PI) for n in range(d // 2)]
        ang = torch.tensor([[float((f[n] * (start + i)) % 1) for n in range(d // 2)] for i in range(s)], dtype=torch.float64) * 2 * math.pi
    y, (a, b) = x.cpu().double(), x.cpu().double().split(d // 2, -1)
    want = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)
    size = (a.abs() + b.abs()).repeat(1, 1, 1, 2)
    rad = 2 * math.pi * (abs(start) / 2 * 2.0 ** -64 + 2.0 ** -33)
    assert ((got.cpu().double() - want).abs() <= size * (rad + math.pi * 2.0 ** -24 + 4 * 2.0 ** -24)).all()
