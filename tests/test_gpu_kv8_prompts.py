"""Attention of whole prompts over the 8-bit cache, every token seeing all before it, against a 64-bit form.

Tolerance as in test_gpu_kv8.attention_ref: a probability may be rounded to f16, a score carries
ds <= (hd + 8) 2^-23 max sum|q||k| scale, so |do| <= 2 (2^-11 + 2 ds) sum p|v| + 2^-8 |o|."""
import math

import pytest
import torch

from glt_b200 import serve
from test_gpu_kv8 import device_error, garbage_cache, i32

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bt,nkv,group,hd,window", [(16, 2, 7, 64, 0), (64, 1, 4, 128, 0), (128, 2, 3, 64, 700), (32, 1, 8, 128, 257)])
def test_a_long_prompt_sees_all_of_itself(bt, nkv, group, hd, window, fmt):
    lens, past = [1777, 640], [0, 301]
    g = torch.Generator(device=DEV).manual_seed(bt + hd)
    maxb = -(-1800 // bt)
    cache = garbage_cache(2 * maxb, bt, nkv, hd, fmt)
    table = torch.randperm(2 * maxb, device=DEV, generator=g).to(torch.int32).view(2, maxb)
    device_error()

    def rows(n, heads):
        return torch.randn(n, heads, hd, device=DEV, generator=g).to(torch.bfloat16)

    cache.append(serve.Kv8Batch(table, i32([0, 0]), past[1], row_start=i32([0, 0, past[1]])), rows(past[1], nkv), rows(past[1], nkv))
    n = sum(lens)
    batch = serve.Kv8Batch(table, i32(past), n, row_start=i32([0, lens[0], n]), max_new=max(lens))
    q = rows(n, nkv * group)
    cache.append(batch, rows(n, nkv), rows(n, nkv))
    o, lse = cache.attention(batch, q, window=window)
    k, v = cache.read(batch, None, max(a + b for a, b in zip(lens, past)))
    at, scale = 0, 1 / math.sqrt(hd)
    for b, (m, p) in enumerate(zip(lens, past)):
        pos, t = p + torch.arange(m, device=DEV), torch.arange(p + m, device=DEV)
        see = t <= pos[:, None]
        if window:
            see &= t > pos[:, None] - window
        for h in range(nkv * group):
            kk, vv, qq = k[b, :p + m, h // group].double(), v[b, :p + m, h // group].double(), q[at:at + m, h].double()
            z = (qq @ kk.t() * scale).masked_fill(~see, -math.inf)
            want_lse = torch.logsumexp(z, -1)
            w = torch.exp(z - want_lse[:, None])
            want = w @ vv
            ds = (qq.abs() @ kk.abs().t()).masked_fill(~see, 0).amax(-1) * scale * (hd + 8) * 2.0 ** -23
            tol = 2 * (2.0 ** -11 + 2 * ds[:, None]) * (w @ vv.abs()) + 2.0 ** -8 * want.abs() + 1e-30
            assert ((o[at:at + m, h].double() - want).abs() <= tol).all()
            ltol = ds + (4 + (p + m) / 32) * 2.0 ** -23 + 2.0 ** -22 * want_lse.abs()
            assert ((lse[at:at + m, h].double() - want_lse).abs() <= ltol).all()
        at += m
    assert device_error() == 0
