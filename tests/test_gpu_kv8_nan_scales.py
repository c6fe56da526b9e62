"""A scale of K that is NaN: rows that see a token of its block get NaN, in o and lse, through every kernel; others do not."""
import math

import pytest
import torch

from test_gpu_kv8_prefix import Case

pytestmark = pytest.mark.gpu
DEV = "cuda"


def only(o, lse, bad):
    """bad [rows, heads]: those are NaN, all else is finite."""
    assert torch.isnan(o[bad]).all() and torch.isnan(lse[bad]).all()
    assert torch.isfinite(o[~bad]).all() and torch.isfinite(lse[~bad]).all()


@pytest.mark.parametrize("fmt,bt,hd", [("int8", 16, 64), ("e4m3", 32, 128), ("int8", 128, 128)])
@pytest.mark.parametrize("rows", [2, 40])
def test_in_the_prefix(fmt, bt, hd, rows):
    c = Case(fmt, bt, 2, 4, hd, 700, [9] * rows, [1] * rows, seed=1)
    for at in (0, 2, 700 // bt):   # the last one is not full
        held = c.ks[c.blocks[at], 1].item()
        c.ks[c.blocks[at], 1] = math.nan
        bad = torch.zeros(rows, 8, dtype=torch.bool, device=DEV)
        bad[:, 4:] = True
        only(*c.run(), bad)
        c.ks[c.blocks[at], 1] = held
    c.check(*c.run())
