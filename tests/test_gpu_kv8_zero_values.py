"""Blocks whose values are all 0 beside others: what they weigh, and nothing else, changes.  Oracle and tolerance of test_gpu_kv8_prefix.py, whose
allowance for small summands goes by the row's largest one among the values that are there."""
import pytest
import torch

from test_gpu_kv8_prefix import Case, take_error

pytestmark = pytest.mark.gpu
DEV = "cuda"


def case(rows, own, seed):
    c = Case("int8", 16, 2, 4, 64, 900, [own] * rows, [1] * rows, seed=seed)
    c.q = c.q.abs()
    return c


def unseen(c, ids):
    """Blocks whose scores lie some hundreds below the others': nothing of their values arrives."""
    c.k[ids.long()] = 1   # -127
    c.ks[ids.long()] *= 20.0


@pytest.mark.parametrize("rows,own", [(3, 20), (50, 20), (50, 400)])
@pytest.mark.parametrize("power", [-89, -75, -7, 20])
def test_beside_scales_of_one_size(rows, own, power):
    c = case(rows, own, 51)
    c.vs *= 2.0 ** (power + 5)
    c.vs[c.blocks.long()[2::3]] = 0.0
    c.vs[c.table[:, 1::2].flatten().long()] = 0.0
    c.check(*c.run())
    assert take_error() == 0


@pytest.mark.parametrize("rows,own", [(3, 20), (50, 20), (50, 400)])
@pytest.mark.parametrize("power", [100, 40, 4])
@pytest.mark.parametrize("first", [0, 1, 20])
def test_beside_a_large_scale_that_does_not_count(rows, own, power, first):
    """Wherever the block with the large scale lies, before the zeros or after them."""
    c = case(rows, own, 52)
    c.vs[c.blocks.long()[2::3]] = 0.0
    c.vs[c.table[:, 1::2].flatten().long()] = 0.0
    for ids in (c.blocks[first:first + 1], c.table[:, 0]):
        unseen(c, ids)
        c.vs[ids.long()] = 2.0 ** power
    c.check(*c.run())
    assert take_error() == 0
