"""Blocks of V whose scales lie so far apart that a token's weight times its scale leaves 32 bits beside another's: its weight
still counts in the sum of weights.

lse does not depend on V.  Exponents here are below 2^8, so that each rounding of one is off by at most 2^-17: the product's, the
reference's sum, one for each move of the reference from one level of scales to another (three at most) and one for each
join (three): 8 * 2^-17 * ln 2 < 2^-14, and 2^-22 |lse| for its own sum."""
import pytest
import torch

from test_gpu_kv8_prefix import Case, take_error

pytestmark = pytest.mark.gpu
DEV = "cuda"

LEVELS = [(100, None), (110, -7, -85), (-89, 30), (110, None, -89)]   # powers of two; None: values of 0


def spread(scales, ids, levels, order):
    """Scales of the blocks `ids` take the levels in turn, or one after the other, up or down."""
    n = len(ids)
    at = torch.arange(n) % len(levels) if order == "turn" else torch.arange(n) * len(levels) // n
    if order == "up":
        at = len(levels) - 1 - at
    for i, lv in enumerate(levels):
        some = ids[(at == i).to(ids.device)].long()
        scales[some] = 0.0 if lv is None else 2.0 ** lv


@pytest.mark.parametrize("rows,own", [(3, 20), (50, 20), (50, 400)])   # 16 rows a KV head or 200; a short table or a long one
@pytest.mark.parametrize("order", ["turn", "down", "up"])
@pytest.mark.parametrize("levels", LEVELS, ids=str)
@pytest.mark.parametrize("where", ["prefix", "own", "both", "apart"])
def test_weights_count_beside_scales_far_away(where, levels, order, rows, own):
    c = Case("int8", 16, 2, 4, 64, 900, [own] * rows, [1] * rows, seed=31)
    _, base = c.run()
    if where in ("prefix", "both"):
        spread(c.vs, c.blocks, levels, order)
    if where in ("own", "both"):
        for b in range(rows):
            spread(c.vs, c.table[b], levels, order)
    if where == "apart":   # the prefix on one level, own tokens on another
        lo, hi = levels[-1], levels[0]
        if order == "up":
            lo, hi = hi, lo
        c.vs[c.blocks.long()] = 0.0 if lo is None else 2.0 ** lo
        c.vs[c.table.flatten().long()] = 0.0 if hi is None else 2.0 ** hi
    o, lse = c.run()
    assert ((lse - base).abs() <= 2.0 ** -14 + 2.0 ** -22 * base.abs()).all(), (lse - base).abs().max()
    c.check(o, base)
    assert take_error() == 0


@pytest.mark.parametrize("levels", LEVELS, ids=str)
def test_weights_count_in_every_part(levels):
    """A long prefix of many parts, several tiles of rows, head_dim 128, e4m3, and rows that see little of the heavy blocks."""
    c = Case("e4m3", 32, 2, 8, 128, 9000, [40, 0, 7], [11, 30, 1], seed=32, q_amp=3.0)
    _, base = c.run()
    spread(c.vs, c.blocks, levels, "turn")
    o, lse = c.run()
    mags = 3.0 * 3.0 * 3.0 * 128 * c.scale * 1.45   # of scores, base 2, at most some: an ulp of 2^-14 below 2^10
    assert mags < 2 ** 10
    assert ((lse - base).abs() <= 2.0 ** -12 + 2.0 ** -22 * base.abs()).all(), (lse - base).abs().max()
    assert torch.isfinite(o).all() and take_error() == 0
