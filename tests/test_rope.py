"""Rotary positions: the table (CPU), refusals (CPU), the kernel against the formulas in 64 bits (GPU)."""
import ctypes
import math

import pytest
import torch

import attn_bwd_b200 as ab
from attn_bwd_b200 import _lib
from fused_reference import HALF_STEP, rope

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _freq(rotary, base=10000.0):
    return base ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)


def _radians(table):
    t = table.turns.cpu()
    return (t.double() % 2.0 ** 64) / 2.0 ** 64 * 2 * math.pi


# ------------------------------------------------------------------ the table
def test_table_frequencies():
    t = ab.rope_table(64, base=500.0, device="cpu")
    assert t.factor == 1.0 and t.turns.dtype == torch.int64
    assert torch.allclose(_radians(t), _freq(64, 500.0), rtol=1e-15, atol=1e-18)
    lin = ab.rope_table(64, base=500.0, scaling={"type": "linear", "factor": 4.0}, device="cpu")
    assert torch.allclose(_radians(lin), _freq(64, 500.0) / 4, rtol=1e-15, atol=1e-18)
    b = ab.rope_table(64, base=500.0, scaling={"type": "base", "factor": 8.0}, device="cpu")
    f = _radians(b)
    assert abs(f[0] - 1) < 1e-14 and abs(f[-1] * 8 / _freq(64, 500.0)[-1] - 1) < 1e-13
    r = ab.rope_table(128, scaling={"type": "ramp", "factor": 8.0, "original_length": 4096}, device="cpu")
    f, f0 = _radians(r), _freq(128)
    turns = 4096 * f0 / (2 * math.pi)
    assert torch.allclose(f[turns > 32], f0[turns > 32]) and torch.allclose(f[turns < 1] * 8, f0[turns < 1])
    assert r.factor == pytest.approx(0.1 * math.log(8.0) + 1)


@pytest.mark.parametrize("args", [(0,), (3,), (-2,), (64, -1.0), (64, 10000.0, {"type": "odd", "factor": 2.0}),
                                  (64, 10000.0, {"type": "linear"}), (64, 10000.0, {"type": "linear", "factor": 0.5}),
                                  (64, 10000.0, {"type": "ramp", "factor": 2.0}), (2, 10000.0, {"type": "base", "factor": 2.0}),
                                  (64, 10000.0, {"type": "linear", "factor": 2.0, "high": 3.0})])
def test_table_refusals(args):
    with pytest.raises(ValueError):
        ab.rope_table(*args, device="cpu")


def test_cpu_tensors_are_refused():
    t = ab.rope_table(64, device="cpu")
    x = torch.zeros(1, 2, 3, 64)
    with pytest.raises(ValueError, match="CUDA"):
        ab.rope_fwd(x, x, torch.arange(3), t)
    with pytest.raises(ValueError):
        ab.rope_fwd(None, None, torch.arange(3), t)
    with pytest.raises(TypeError):
        ab.rope_fwd(x, x, torch.arange(3), None)


@pytest.mark.parametrize("bad,code", [(dict(bs=-1), 1), (dict(seq=-1), 1), (dict(rotary_dim=3), 1), (dict(rotary_dim=0), 1),
                                      (dict(rotary_dim=256), 1), (dict(head_dim=5000), 1), (dict(q_heads=-1), 1),
                                      (dict(position_stride=-1), 1), (dict(dtype=7), 3)])
def test_c_entry_refuses_without_device(bad, code):
    a = _lib.RopeArgs()
    base = dict(bs=1, seq=4, q_heads=2, k_heads=1, head_dim=128, rotary_dim=128, dtype=0, factor=1.0, position_stride=0)
    base.update(bad)
    for n, x in base.items():
        setattr(a, n, x)
    lib = _lib.load()
    assert lib.attn_bwd_b200_rope(ctypes.byref(a), 16, 16, 16, 16, 16, 16, 0) == code
    assert lib.attn_bwd_b200_rope(None, 16, 16, 16, 16, 16, 16, 0) == _lib.EINVAL


# ------------------------------------------------------------------ the kernel
def _states(bs, h, kv, s, d, dtype, seed=0, bshd=True):
    g = torch.Generator().manual_seed(seed)
    mk = lambda n: torch.randn(bs, s, n, d, generator=g).to(dtype).cuda().transpose(1, 2)
    q, k = mk(h), mk(kv)
    return (q, k) if bshd else (q.contiguous(), k.contiguous())


def _check(got, x, pos, freq, rotary, **kw):
    want = rope(x.cpu(), pos.cpu(), freq, rotary, **kw)
    # the rounding of the result, and 4 half steps of fp32 on each of the two products
    size = rope(x.cpu().double().abs(), torch.zeros_like(pos).cpu(), freq, rotary, interleaved=kw.get("interleaved", False))
    n = rotary // 2
    a = x.cpu().double().abs()[..., :rotary]
    pair = (a.unflatten(-1, (n, 2)).flip(-1).flatten(-2) if kw.get("interleaved") else torch.cat([a[..., n:], a[..., :n]], -1))
    size[..., :rotary] += pair
    tol = HALF_STEP[x.dtype] * want.abs() + 4 * 2.0 ** -24 * size * abs(kw.get("factor", 1.0)) + (2.0 ** -25 if x.dtype == HF else 0)
    err = (got.cpu().double() - want).abs()
    assert (err <= tol).all(), float((err - tol).max())
    assert torch.equal(got[..., rotary:], x[..., rotary:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("bs,h,kv,s,d,rotary", [(2, 80, 8, 5, 128, 128), (1, 3, 1, 33, 64, 32), (3, 4, 4, 1, 80, 80),
                                                (1, 2, 1, 7, 96, 10), (2, 5, 1, 9, 6, 2), (1, 1, 1, 1, 2, 2),
                                                (1, 2, 2, 3, 4096, 4096), (1, 300, 1, 2, 256, 128)])
def test_rotation_and_gradient(cuda, bs, h, kv, s, d, rotary, interleaved, dtype):
    for bshd in (True, False):
        q, k = _states(bs, h, kv, s, d, dtype, bshd=bshd)
        table, freq = ab.rope_table(rotary), _freq(rotary)
        pos = torch.randint(0, 5000, (bs, s), generator=torch.Generator().manual_seed(1)).cuda()
        for fn, inverse in ((ab.rope_fwd, False), (ab.rope_bwd, True)):
            for x, y in zip((q, k), fn(q, k, pos, table, interleaved=interleaved)):
                assert y.shape == x.shape and y.dtype == x.dtype
                _check(y, x, pos, freq, rotary, interleaved=interleaved, inverse=inverse)


@pytest.mark.gpu
def test_far_positions_and_position_forms(cuda):
    q, k = _states(2, 3, 1, 4, 128, F32)
    table, freq = ab.rope_table(128), _freq(128)
    far = torch.tensor([0, 1 << 20, (1 << 30) + 12345, -7], device="cuda")
    for pos in (far, far[None], far.to(torch.int32), torch.stack([far, far + 3])):
        got, _ = ab.rope_fwd(q, k, pos, table)
        # float64 angles of the reference itself: pos * 2^-53
        assert (got.cpu().double() - rope(q.cpu(), pos.cpu(), freq, 128)).abs().max() < 2e-6
    one, _ = ab.rope_fwd(q, None, far, table)
    assert torch.equal(one, ab.rope_fwd(q, k, far, table)[0])
    none, two = ab.rope_fwd(None, k, far, table)
    assert none is None and torch.equal(two, ab.rope_fwd(q, k, far, table)[1])


@pytest.mark.gpu
def test_offsets_above_32_bits(cuda):
    """17 million positions of one head: the last rows are what a short call gives for them."""
    n = 17_000_003
    k = torch.empty(1, 1, n, 128, dtype=BF, device="cuda").normal_()
    table, pos = ab.rope_table(128), torch.arange(n, device="cuda")
    _, got = ab.rope_fwd(None, k, pos, table)
    for part in (slice(0, 70), slice(8_388_600, 8_388_700), slice(n - 50, n)):
        assert torch.equal(got[:, :, part], ab.rope_fwd(None, k[:, :, part], pos[part], table)[1])


@pytest.mark.gpu
def test_scaled_table_and_gradient_against_differences(cuda):
    scaling = {"type": "ramp", "factor": 8.0, "original_length": 64, "low": 1.0, "high": 8.0}
    table = ab.rope_table(64, scaling=scaling)
    q, k = _states(1, 2, 1, 6, 64, F32)
    pos = torch.arange(6, device="cuda") + 1000
    freq = _radians(table)
    got, _ = ab.rope_fwd(q, k, pos, table)
    _check(got, q, pos, freq, 64, factor=table.factor)
    g, step = torch.randn_like(q), torch.randn_like(q)
    dq, _ = ab.rope_bwd(g, k, pos, table)
    f = lambda x: (rope(x, pos.cpu(), freq, 64, factor=table.factor) * g.cpu().double()).sum()
    diff = (f(q.cpu().double() + 1e-4 * step.cpu()) - f(q.cpu().double() - 1e-4 * step.cpu())) / 2e-4
    assert abs(diff - (dq.cpu().double() * step.cpu().double()).sum()) < 1e-4 * (1 + abs(diff))


@pytest.mark.gpu
def test_in_place_strides_streams_and_graphs(cuda):
    q, k = _states(2, 6, 2, 37, 64, BF)
    table = ab.rope_table(48)
    pos = torch.arange(37, device="cuda")
    a, b = ab.rope_fwd(q, k, pos, table)
    assert a.stride() == q.stride() and b.stride() == k.stride()
    q2, k2 = q.clone(), k.clone()
    r = ab.rope_fwd(q2, k2, pos, table, out=(q2, k2))
    assert r[0] is q2 and torch.equal(q2, a) and torch.equal(k2, b)
    wide = torch.zeros(2, 6, 37, 67, dtype=BF, device="cuda")   # rows at odd addresses, neighbours kept
    wide[..., 3:] = q
    out = torch.full((2, 6, 37, 70), 7.0, dtype=BF, device="cuda")
    ab.rope_fwd(wide[..., 3:], None, pos, table, out=(out[..., 1:65], None))
    assert torch.equal(out[..., 1:65], a) and (out[..., :1] == 7).all() and (out[..., 65:] == 7).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c, _ = ab.rope_fwd(q, k, pos, table)
    side.synchronize()
    assert torch.equal(c, a)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        d, _ = ab.rope_fwd(q2, k2, pos, table)
    q2.copy_(q)
    g.replay()
    assert torch.equal(d, a)
    back, _ = ab.rope_bwd(a.float(), b.float(), pos, table)
    assert (back - q.float()).abs().max() < 0.03   # two bf16 half steps of values below 4.2


@pytest.mark.gpu
def test_python_refusals(cuda):
    q, k = _states(2, 4, 2, 5, 64, BF)
    t, pos = ab.rope_table(64), torch.arange(5, device="cuda")
    for args in ((q, k[:1], pos, t), (q, k[..., :32], pos, t), (q, k, pos[:4], t), (q, k, pos.cpu(), t),
                 (q, k, pos, ab.rope_table(128)), (q, k, pos, ab.rope_table(64, device="cpu")), (q[0], k[0], pos, t),
                 (q, k.float(), pos, t)):
        with pytest.raises(ValueError):
            ab.rope_fwd(*args)
    for args in ((q, k, pos.float(), t), (q.double(), k.double(), pos, t)):
        with pytest.raises(TypeError):
            ab.rope_fwd(*args)
    for out in ((q,), (q.float(), k), (q[:1], k), (q[..., :1, :].expand_as(q), k)):
        with pytest.raises(ValueError):
            ab.rope_fwd(q, k, pos, t, out=out)
    empty = ab.rope_fwd(q[:, :, :0], k[:, :, :0], pos[:0], t)
    assert empty[0].shape == (2, 4, 0, 64)
