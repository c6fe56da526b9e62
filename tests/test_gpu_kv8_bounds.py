"""`max_new` is a bound: one that says no more than the rows and the table do gives the same results."""
import pytest
import torch

from glt_b200 import serve
from test_gpu_kv8 import attention_ref, check, device_error, garbage_cache, i32

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("max_new", [37, 45, 1000, 2 ** 30, 2 ** 31 - 200, 2 ** 31 - 1])
@pytest.mark.parametrize("bt", [16, 128])
def test_any_bound_that_holds(bt, max_new):
    g = torch.Generator(device=DEV).manual_seed(bt)
    rows, past, starts = 45, [3, 0, 70], [0, 37, 38, 45]
    k, v = torch.randn(2, rows, 2, 64, device=DEV, generator=g).to(torch.bfloat16)
    q = torch.randn(rows, 8, 64, device=DEV, generator=g).to(torch.bfloat16)
    old = torch.randn(73, 2, 64, device=DEV, generator=g).to(torch.bfloat16)
    table = torch.arange(24, device=DEV, dtype=torch.int32).view(3, 8)
    device_error()

    def run(bound):
        cache = garbage_cache(24, bt, 2, 64, "int8")
        cache.append(serve.Kv8Batch(table, i32([0, 0, 0]), 73, row_start=i32([0, 3, 3, 73]), max_new=70), old, old)
        batch = serve.Kv8Batch(table, i32(past), rows, row_start=i32(starts), max_new=bound)
        cache.append(batch, k, v)
        return (*cache.read(batch, None, 80), *cache.attention(batch, q))

    want_k, want_v, _, _ = run(37)
    got_k, got_v, o, lse = run(max_new)
    assert torch.equal(got_k, want_k) and torch.equal(got_v, want_v)
    for b in range(3):
        sl, n = slice(starts[b], starts[b + 1]), past[b] + starts[b + 1] - starts[b]
        ref = attention_ref(q[sl].cpu(), want_k[b, :n].cpu().double(), want_v[b, :n].cpu().double(), past[b], 0.125)
        check(o[sl], lse[sl], ref, f"sequence {b}")
    assert device_error() == 0
