"""Rows of any size through the norm of the 8-bit quantisation, against the formula in 64 bits.

The tolerance is that of test_gpu_w8.test_codes_of_a_norm: a value is off by some 70 * 2^-24 whatever its row's size, a
quotient of up to 127 by 127 * 140 * 2^-24, so that only quotients as near as that to k + 1/2 may have the other code."""
import math

import pytest
import torch

from glt_b200 import serve

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOP = torch.finfo(torch.bfloat16).max
LENGTHS = [2, 300, 4096, 5000, 14336, 20001]   # rows in two vectors a thread, in four, and read again for each pass


def check(x, eps, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    K = x.shape[1]
    w = (1 + 0.3 * torch.randn(K, device=DEV, generator=g)).to(torch.bfloat16)
    q = serve.quantize_rows(x, w, eps)
    eps = torch.tensor(eps, dtype=torch.float32).double().item()   # as the call takes it
    y = x.double() / torch.sqrt(x.double().square().mean(1, keepdim=True) + eps) * w.double()
    s = y.abs().amax(1) / 127
    off = 70 * 2.0 ** -24
    assert ((q.scales.double() - s).abs() <= 2 * off * s).all(), (q.scales, s)
    quot = torch.where(s[:, None] > 0, y / s[:, None], torch.zeros_like(y))
    assert ((q.codes.double() - quot).abs() <= 0.5 + 127 * 2 * off).all()


def randn(K, seed, rows=3):
    return torch.randn(rows, K, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))


@pytest.mark.parametrize("K", LENGTHS)
@pytest.mark.parametrize("amp", [1e19, 1e30, 1e36, 1e37, math.inf])
def test_large_rows(K, amp):
    """Sums of squares beyond 32 bits, up to rows of nothing but the type's largest values."""
    x = randn(K, K)
    x = (torch.sign(x) * TOP if amp == math.inf else (x * amp).clamp(-TOP, TOP)).to(torch.bfloat16)
    assert torch.isfinite(x).all()
    check(x, 1e-6, K)
    x[1, 1:] = 0.5   # one large value among small ones
    x[1, 0] = TOP
    check(x, 0.0, K)


@pytest.mark.parametrize("amp,eps", [(1e19, 3e38), (1.0, 3e38), (1.5e19, 1e38)])
def test_large_eps(amp, eps):
    check((randn(700, 1).clamp(-1.5, 1.5) * amp).to(torch.bfloat16), eps)


def test_rows_that_hold_an_infinity_or_nan_have_no_scale():
    x = randn(600, 2, 5).to(torch.bfloat16)
    x[1, 7], x[2, 599], x[3, 0] = math.inf, -math.inf, math.nan
    x[2, :300] = TOP
    q = serve.quantize_rows(x, torch.ones(600, device=DEV, dtype=torch.bfloat16))
    assert torch.isnan(q.scales[1:4]).all() and (q.codes[1:4] == 0).all() and torch.isfinite(q.scales[[0, 4]]).all()
