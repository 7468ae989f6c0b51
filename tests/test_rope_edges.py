"""Rotary positions: tables and results that a caller makes itself."""
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
