"""A prefix without blocks holds no token: another length is reported, and counts as none."""
import pytest

import torch

from test_gpu_kv8_prefix import Case, take_error

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("own", [30, 600], ids=["short", "long"])
@pytest.mark.parametrize("length", [1, 5, -1, 2 ** 31 - 1, -2 ** 31])
def test_length_without_blocks(own, length):
    c = Case("int8", 16, 2, 4, 64, 0, [own, 3], [1, 1], seed=41)
    take_error()
    assert c.blocks.numel() == 0
    want = c.run()
    assert take_error() == 0
    c.length.fill_(length)
    o, lse = c.run()
    assert take_error() == 2
    c.check(o, lse)
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
