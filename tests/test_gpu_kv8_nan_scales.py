"""A scale of K that is NaN: rows that see a token of its block get NaN, in o and lse, through every kernel; others do not."""
import math

import pytest
import torch

from glt_b200 import serve
from test_gpu_kv8_prefix import Case, take_error

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


@pytest.mark.parametrize("own", [40, 400], ids=["short", "long"])
@pytest.mark.parametrize("fmt,bt,hd", [("int8", 16, 64), ("e4m3", 32, 128), ("e4m3", 16, 128)])
def test_among_own_tokens(fmt, bt, hd, own):
    c = Case(fmt, bt, 2, 4, hd, 100, [own, own, 5], [1, 3, 2], seed=2)
    c.ks[c.table[1, 1], 0] = math.nan
    bad = torch.zeros(6, 8, dtype=torch.bool, device=DEV)
    bad[1:4, :4] = True
    only(*c.run(), bad)
    # masked, the block is not seen
    c.mask = torch.ones(3, c.table.shape[1] * bt, device=DEV, dtype=torch.uint8)
    c.mask[1, bt:2 * bt] = 0
    c.check(*c.run())
    assert take_error() == 0


@pytest.mark.parametrize("window,sinks", [(0, 0), (60, 0), (60, 5)])
@pytest.mark.parametrize("fmt,bt,hd,group", [("int8", 16, 64, 4), ("e4m3", 32, 128, 4), ("e4m3", 16, 128, 8), ("int8", 64, 64, 8)])
@pytest.mark.parametrize("new", [1, 5])
def test_without_a_prefix(fmt, bt, hd, group, new, window, sinks):
    c = Case(fmt, bt, 2, group, hd, 0, [300] * 2, [new] * 2, seed=3)
    cache, batch, _, _ = c.objects()
    none = torch.zeros(2 * new, 2 * group, dtype=torch.bool, device=DEV)
    for at, seen in ((0, window == 0 or sinks > 0), (150 // bt, window == 0), (290 // bt, True)):
        held = c.ks[c.table[0, at], 1].item()
        c.ks[c.table[0, at], 1] = math.nan
        bad = none.clone()
        bad[:new, group:] = seen
        only(*cache.attention(batch, c.q, window=window, sinks=sinks), bad)
        mask = torch.ones(2, c.table.shape[1] * bt, device=DEV, dtype=torch.uint8)
        mask[0, at * bt:(at + 1) * bt] = 0
        only(*cache.attention(batch, c.q, window=window, sinks=sinks, token_mask=mask), none)
        c.ks[c.table[0, at], 1] = held
