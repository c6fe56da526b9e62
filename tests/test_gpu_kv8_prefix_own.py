"""Own tokens behind a shared prefix: short tables, which one kernel takes whole, and long ones, which are split.

The oracle and its tolerance are those of test_gpu_kv8_prefix.py; a weight of the short tables' kernel below f16's normal
range is off by at most half of 2^-24 where the running maximum counts 2^15, so within 2^-40 of the largest
summand, less than is allowed there."""
import math

import pytest
import torch

from test_gpu_kv8_prefix import Case, take_error

pytestmark = pytest.mark.gpu
DEV = "cuda"

SHAPES = [  # fmt, bt, nkv, group, hd, prefix, own, news
    ("int8", 16, 3, 5, 64, 100, [255, 0, 1, 15, 16, 17], [1] * 6),             # 256 tokens a table, rows of no full tile
    ("e4m3", 128, 2, 4, 128, 300, [255, 128, 127], [1] * 3),
    ("int8", 64, 1, 1, 128, 70, [219, 3], [37, 20]),                           # 37 rows a KV head
    ("e4m3", 16, 5, 3, 64, 33, [30, 0, 9], [7, 0, 23]),                        # five KV heads over warps of four
    ("int8", 32, 1, 16, 64, 64, [5] * 4, [1] * 4),                             # a tile exactly
    ("e4m3", 32, 2, 17, 128, 64, [5] * 4, [1] * 4),                            # and one row more
    ("int8", 128, 2, 8, 64, 0, [60, 61], [3, 3]),                              # a prefix without tokens
    ("int8", 16, 3, 5, 64, 100, [256, 0, 1, 300], [1] * 4),                    # longer tables
    ("e4m3", 128, 2, 4, 128, 300, [700, 128, 3], [1] * 3),
    ("int8", 64, 1, 3, 128, 70, [500, 3], [37, 20]),
    ("e4m3", 16, 5, 3, 64, 33, [400, 0, 9], [7, 0, 23]),
    ("int8", 32, 2, 8, 64, 0, [1000, 61], [3, 3]),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_matches_the_formula(shape):
    c = Case(*shape, seed=len(str(shape)) + 100)
    c.check(*c.run())
    assert take_error() == 0


LENGTHS = [pytest.param([40, 12, 0], id="short"), pytest.param([400, 12, 0], id="long")]


@pytest.mark.parametrize("own", LENGTHS)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("hd", [64, 128])
def test_masked_and_unseen_tokens_may_hold_anything(fmt, hd, own):
    c = Case(fmt, 16, 2, 3, hd, 70, own, [3, 3, 3], seed=21)
    room = c.table.shape[1] * 16
    g = torch.Generator(device=DEV).manual_seed(22)
    c.mask = (torch.rand(3, room, device=DEV, generator=g) < 0.6).to(torch.uint8)
    c.mask[0, 16:32] = 0   # a block of which nothing is seen
    c.mask[1] = 0          # and a sequence
    want = c.run()
    c.check(*want)
    for b in range(3):
        total = c.own[b] + 3
        for t in range(room):
            if t >= total or not c.mask[b, t]:
                i = int(c.table[b, t // 16])
                c.k[i, :, t % 16] = c.v[i, :, t % 16] = 0xFF if fmt == "e4m3" else 0
        for blk in range(room // 16):
            if blk * 16 >= total or not c.mask[b, blk * 16:min(total, blk * 16 + 16)].any():
                c.ks[c.table[b, blk]] = c.vs[c.table[b, blk]] = math.nan
    got = c.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert take_error() == 0


@pytest.mark.parametrize("own", LENGTHS)
def test_bad_own_blocks_are_skipped(own):
    c = Case("int8", 16, 2, 4, 64, 50, own, [2, 2, 2], seed=23)
    take_error()
    good = c.table.clone()
    for bad in (-1, c.k.shape[0], 2 ** 31 - 1, -2 ** 31):
        c.table[0, 1] = bad
        o, lse = c.run()
        c.table.copy_(good)
        assert take_error() == 2
        c.mask = torch.ones(3, c.table.shape[1] * 16, device=DEV, dtype=torch.uint8)
        c.mask[0, 16:32] = 0
        c.check(o, lse)
        c.mask = None
    c.check(*c.run())
    assert take_error() == 0


@pytest.mark.parametrize("own", LENGTHS)
@pytest.mark.parametrize("spread", [0.0, 15.0])
def test_own_values_of_very_different_scales(own, spread):
    c = Case("e4m3", 16, 2, 3, 128, 90, own, [5, 5, 5], seed=24, spread=spread)
    c.vs[c.table[0, ::2].long()] = 0.0
    c.check(*c.run())
    c.length.zero_()
    c.check(*c.run(), pre=0)


@pytest.mark.parametrize("own", LENGTHS)
def test_a_nan_query_stays_in_its_row(own):
    c = Case("int8", 32, 2, 4, 64, 40, own, [2, 2, 2], seed=25)
    c.q = c.q.clone()
    c.q[1, 3, 7] = math.nan
    c.q[2, 0] = 0
    o, lse = c.run()
    bad = torch.zeros(o.shape[:2], dtype=torch.bool, device=DEV)
    bad[1, 3] = True
    assert torch.isnan(o[bad]).all() and torch.isfinite(o[~bad]).all()
    assert torch.isnan(lse[bad]).all() and torch.isfinite(lse[~bad]).all()
