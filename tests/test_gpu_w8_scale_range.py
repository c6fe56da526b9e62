"""8-bit products whose sum times the channel's scale alone would leave 32 bits, though the result does not; the oracle and its
tolerance are test_gpu_w8's."""
import pytest
import torch

from glt_b200 import serve
from test_gpu_w8 import DEV, codes_ref, gen, near, product_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(1, 200, 5000), (5, 300, 384), (70, 333, 1024), (700, 300, 384), (300, 37900, 130)])
@pytest.mark.parametrize("out,resid", [(torch.bfloat16, False), (torch.float32, True)])
def test_large_channel_scales(M, N, K, out, resid):
    g = gen(M)
    x = (torch.randn(M, K, device=DEV, generator=g) * torch.logspace(-30, -25, M, device=DEV)[:, None]).to(torch.bfloat16)
    codes = torch.randint(-127, 128, (N, K), device=DEV, generator=g, dtype=torch.int8)
    # weights of up to bf16's largest value, 3.4e38: scales of up to 2.67e36
    scales = torch.logspace(20, 36.42, N, device=DEV)[torch.randperm(N, device=DEV, generator=g)]
    w = serve.W8Weight.from_codes(codes, scales)
    r = torch.randn(M, N, device=DEV, generator=g).to(torch.bfloat16) if resid else None
    c, s = codes_ref(x.float())
    want, tol = product_ref(c, s, codes, scales, r)
    assert (want.abs() < 3e38).all() and ((c.double() @ codes.double().t()).abs() * scales.double()).max() > 3.4e38
    near(w.linear(x, resid=r, out_dtype=out), want, tol)
