"""Rows whose squares are below 32 bits, through the norm of the 8-bit quantisation; tolerance as in test_gpu_w8_norm_range."""
import pytest
import torch

from glt_b200 import serve
from test_gpu_w8_norm_range import DEV, LENGTHS, check, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K", LENGTHS)
@pytest.mark.parametrize("amp,eps", [(1e-14, 0.0), (1e-18, 0.0), (1e-20, 0.0), (1e-25, 0.0), (1e-38, 0.0), (3e-40, 0.0),
                                     (1e-20, 1e-39), (1e-23, 1e-45), (1e-18, 1e-36), (1e-25, 1e-30)])
def test_small_rows(K, amp, eps):
    x = (randn(K, K) * amp).to(torch.bfloat16)
    assert (x != 0).any(1).all()
    check(x, eps, K)


def test_zeros():
    """With eps 0 a row of zeros is 0 / 0."""
    x = torch.zeros(2, 500, device=DEV, dtype=torch.bfloat16)
    x[1] = 1
    norm = torch.ones(500, device=DEV, dtype=torch.bfloat16)
    for eps in (1e-6, 1e-38, 1e-45):
        q = serve.quantize_rows(x, norm, eps)
        assert q.scales[0] == 0 and (q.codes[0] == 0).all() and (q.codes[1] == 127).all()
    q = serve.quantize_rows(x, norm, 0.0)
    assert torch.isnan(q.scales[0]) and (q.codes[0] == 0).all() and (q.codes[1] == 127).all()
