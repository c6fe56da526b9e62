"""Prompts of hundreds of new tokens a sequence: behind a shared prefix, and with a window and first tokens.  Oracles and tolerances are those
of test_gpu_kv8_prefix.py and test_gpu_kv8_window.py."""
import pytest
import torch

import test_gpu_kv8_prefix as prefix
import test_gpu_kv8_window as window

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,bt,nkv,group,hd,pre,own,news", [
    ("int8", 16, 2, 3, 64, 1000, [0, 0], [300, 300]),
    ("e4m3", 64, 1, 4, 128, 333, [0, 130, 7], [513, 1, 200]),
    ("int8", 128, 2, 7, 64, 65, [0], [700]),
    ("e4m3", 32, 1, 1, 128, 0, [5, 0], [257, 300]),
], ids=str)
def test_prompts_behind_a_prefix(fmt, bt, nkv, group, hd, pre, own, news):
    c = prefix.Case(fmt, bt, nkv, group, hd, pre, own, news, seed=pre)
    c.check(*c.run())
    assert prefix.take_error() == 0


@pytest.mark.parametrize("fmt,bt,nkv,group,hd,lens,new,size,first", [
    ("int8", 16, 2, 3, 64, [0, 0, 77], 300, 40, 5),
    ("e4m3", 64, 1, 4, 128, [0, 500], 420, 129, 67),
    ("int8", 128, 2, 7, 64, [3], 513, 256, 4),
    ("e4m3", 16, 1, 1, 128, [0, 1000], 257, 1, 1),
    ("int8", 32, 1, 5, 64, [0, 50], 300, 700, 31),
], ids=str)
def test_prompts_with_a_window(fmt, bt, nkv, group, hd, lens, new, size, first):
    c = window.Case(fmt, bt, nkv, group, hd, lens, new, size, first, seed=new)
    window.take_error()
    c.check(*c.run())
    assert window.take_error() == 0


def test_masked_prompts_with_a_window():
    c = window.Case("e4m3", 32, 2, 2, 64, [0, 90, 400], 260, 100, 20, seed=9, masked=True)
    c.check(*c.run())
