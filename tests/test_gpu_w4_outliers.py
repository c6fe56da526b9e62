"""Products with 4-bit weights where a few columns of x are far larger than the others, as activations of
language models have them: y[m, n] = sum_k x[m, k] s[n, k / G] (u[n, k] - z[n, k / G]).

Tolerance, from the formula alone: x and the codes are exact, so 32-bit sums of K terms, truncated inside the
tensor core, give at most (8 * 2^-22 + (K/32 + 16) * 2^-23) * sum |x||w|; where the outlier's own weight is 0 it is no
part of that.  Beside it each element may lose what lies below 2^-30 of the largest of its 128 columns.  An output in
bf16 lies between the bf16 numbers nearest to the ends of that range: rounding keeps the order."""
import pytest
import torch

from glt_b200 import serve

pytestmark = pytest.mark.gpu
DEV = "cuda"


def weight(N, K, group, asym, zero_at, g):
    """Codes with a weight of exactly 0 in the columns of `zero_at` for all rows but every eighth."""
    codes = torch.randint(0, 16, (N, K), device=DEV, generator=g).to(torch.uint8)
    s = (torch.rand(N, K // group, device=DEV, generator=g) * 0.02 + 0.001).to(torch.bfloat16)
    z = torch.randint(0, 16, s.shape, device=DEV, generator=g).to(torch.uint8) if asym else torch.full_like(s, 8).to(torch.uint8)
    full = z.repeat_interleave(group, 1)
    rows = torch.arange(N, device=DEV) % 8 != 0
    for k in zero_at:
        codes[rows, k] = full[rows, k]
    w = ((codes.double() - full.double()) * s.double().repeat_interleave(group, 1))
    return serve.W4Weight.from_codes(codes, s, z if asym else None), w


def check(y, x, w, K, group, resid=None):
    xd, ad = x.double(), x.double().abs()
    ref = xd @ w.t()
    tol = (ad @ w.abs().t()) * (8 * 2.0 ** -22 + (K / 32 + 16) * 2.0 ** -23) + 1e-30
    pad = -K % 128
    peak = torch.nn.functional.pad(ad, (0, pad)).view(x.shape[0], -1, 128).amax(-1).repeat_interleave(128, 1)[:, :K]
    tol = tol + 2.0 ** -30 * peak @ w.abs().t()
    if resid is not None:
        ref = ref + resid.double()
        tol = tol + ref.abs() * 2.0 ** -23
    low, high = ((ref + d).float().to(y.dtype) for d in (-tol, tol))
    assert ((low <= y) & (y <= high)).all(), ((y.double() - ref).abs() / tol).max().item()


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("times", [1000.0, 3000.0, 2.0 ** 14, 1e6])
@pytest.mark.parametrize("M,group,asym", [(1, 128, False), (2, 32, True), (3, 64, False), (8, 128, True), (9, 32, False),
                                          (16, 64, True), (19, 32, True), (24, 128, False), (32, 64, False), (41, 32, True)])
def test_one_strong_channel_in_128(M, group, asym, times, out):
    N, K = 200, 1152
    g = torch.Generator(device=DEV).manual_seed(M + group)
    strong = [5 + 128 * i + 17 * (i % 3) for i in range(9)]
    w, values = weight(N, K, group, asym, strong, g)
    x = torch.randn(M, K, device=DEV, generator=g)
    x[:, strong] *= times
    x = x.to(torch.bfloat16)
    check(w.linear(x, out_dtype=out), x, values, K, group)


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mantissa", [1.0, 1.0078125, 1.984375, 1.9921875])
@pytest.mark.parametrize("M", [1, 2, 5, 17, 30])
def test_largest_magnitudes_of_every_kind(M, mantissa, out):
    """Blocks whose largest magnitude is a power of two, the largest mantissa or next to either, at any exponent, the
    other columns up to 2^14 below it."""
    N, K, group = 72, 896, 32
    g = torch.Generator(device=DEV).manual_seed(M)
    top = torch.arange(7, device=DEV) + 128 * torch.arange(7, device=DEV)
    w, values = weight(N, K, group, M % 2 == 0, top.tolist(), g)
    x = torch.randn(M, K, device=DEV, generator=g).clamp(-3.9, 3.9)
    for i, e in enumerate((0, 100, -100, 30, -60, 3, -17)):
        part = x[:, 128 * i:128 * i + 128]
        part *= 2.0 ** (e - torch.randint(2, 15, part.shape, device=DEV, generator=g).float())
        part[:, top[i] - 128 * i] = mantissa * 2.0 ** e * (1 - 2 * (i % 2))
    x = x.to(torch.bfloat16)
    check(w.linear(x, out_dtype=out), x, values, K, group)


@pytest.mark.parametrize("M", [1, 4, 20])
def test_subnormal_rows_and_large_scales(M):
    """Rows of bf16's smallest numbers, whose products are ordinary ones under large scales."""
    N, K, group = 40, 256, 64
    g = torch.Generator(device=DEV).manual_seed(M)
    codes = torch.randint(0, 16, (N, K), device=DEV, generator=g).to(torch.uint8)
    s = (torch.rand(N, K // group, device=DEV, generator=g) * 2.0 ** 120).to(torch.bfloat16)
    values = (codes.double() - 8) * s.double().repeat_interleave(group, 1)
    x = torch.randint(-127, 128, (M, K), device=DEV, generator=g).double() * 2.0 ** -133
    x = x.to(torch.bfloat16)
    y = serve.W4Weight.from_codes(codes, s).linear(x, out_dtype=torch.float32)
    assert y.abs().max() > 1e-4
    check(y, x, values, K, group)


def test_a_strong_channel_with_a_residual_and_strides():
    N, K, group, M = 264, 1024, 128, 21
    g = torch.Generator(device=DEV).manual_seed(1)
    w, values = weight(N, K, group, True, [100, 600], g)
    x = torch.randn(M, K + 8, device=DEV, generator=g)
    x[:, [100, 600]] *= 2000
    x = x.to(torch.bfloat16)[:, :K]
    r = torch.randn(M, N, device=DEV, generator=g).to(torch.bfloat16)
    check(w.linear(x, resid=r), x, values, K, group, r)
