"""Attention over the 8-bit cache where the block table holds blocks that no query sees: before every query's
window, or hidden by the token mask.  Nothing in them counts: codes that are NaN patterns, scales that are NaN
or infinite, and, before the window, ids outside the pool.  Results are held to the 64-bit form's tolerances
(test_gpu_kv8.attention_ref), and the error word stays 0."""
import math

import pytest
import torch

from test_gpu_kv8 import Session, device_error

pytestmark = pytest.mark.gpu


def session(fmt, bt, nkv, group, hd, lens, scale):
    s = Session(fmt, bt, nkv, group, hd, seqs=len(lens), room=max(lens) + 40, seed=bt + hd + group)
    device_error()
    s.step(lens, window=1)
    used = set(s.table.flatten().tolist())
    spare = [i for i in range(s.cache.num_blocks) if i not in used]
    for i in spare:
        for t in (s.cache.k, s.cache.v):
            t[i] = 0xFF if fmt == "e4m3" else 0
        for t in (s.cache.k_scale, s.cache.v_scale):
            t[i] = scale
    return s, spare


@pytest.mark.parametrize("scale", [math.nan, math.inf])
@pytest.mark.parametrize("dropped", ["unwritten", "outside"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bt,nkv,group,hd", [(16, 2, 4, 64), (16, 1, 8, 128), (32, 2, 3, 64), (64, 1, 4, 128)])
@pytest.mark.parametrize("new,window", [(1, 33), (1, 1), (1, 47), (5, 20), (3, 64)])
def test_blocks_before_the_window(bt, nkv, group, hd, new, window, fmt, dropped, scale):
    lens = [150, 61, 96, 111]
    s, spare = session(fmt, bt, nkv, group, hd, lens, scale)
    for b, past in enumerate(lens):
        first = past - window + 1            # the oldest token that any query sees
        for k in range(max(first, 0) // bt):
            s.table[b, k] = spare[k % len(spare)] if dropped == "unwritten" else (-1 if k % 2 else s.cache.num_blocks)
    s.step([new] * len(lens), window=window)


@pytest.mark.parametrize("scale", [math.nan, math.inf])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bt,nkv,group,hd", [(16, 2, 4, 64), (16, 1, 8, 128), (32, 2, 7, 64), (64, 1, 4, 128), (128, 1, 2, 64)])
@pytest.mark.parametrize("new", [1, 4])
def test_blocks_that_the_mask_hides(bt, nkv, group, hd, new, fmt, scale):
    """Hidden blocks first (as padding on the left leaves them), in the middle, and all of them."""
    lens = [3 * bt + 7, 4 * bt, 2 * bt + 1, 2 * bt]
    s, spare = session(fmt, bt, nkv, group, hd, lens, scale)
    mask = torch.ones(len(lens), s.maxb * bt, dtype=torch.uint8)
    for b, blocks in enumerate(([0], [1, 2], [0, 1], [0, 1])):
        for k in blocks:
            s.table[b, k] = spare[k]
            mask[b, k * bt:(k + 1) * bt] = 0
    mask[3] = 0
    s.step([new] * len(lens), mask=mask)
