"""4-bit weights (glt_w4_quantize / pack / unpack / linear) against 64-bit forms.

Quantisation is held to equality (the scale is a bf16 rounding of a 32-bit
quotient, the code the nearest to a 32-bit quotient).  A product's tolerance:
32-bit sums of K terms, truncated inside the tensor core, give at most
(8 * 2^-22 + (K/32 + 16) * 2^-23) * sum |x||w|; bf16 output adds 2^-9 |y|."""
import math

import pytest
import torch

from glt_b200 import serve

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ref_quantize(w, group, asym):
    N, K = w.shape
    x = torch.nan_to_num(w.double(), nan=0.0, posinf=math.inf, neginf=-math.inf).view(N, -1, group)
    fin = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    lo, hi = fin.amin(-1).clamp(max=0), fin.amax(-1).clamp(min=0)
    if asym:
        s = ((hi - lo).float().double() / 15).float().to(torch.bfloat16)
        z = torch.where(s > 0, (-lo / s.double()).float().round().clamp(0, 15), torch.zeros_like(lo).float())
    else:
        s = (torch.maximum(hi, -lo) / 7).float().to(torch.bfloat16)
        z = torch.full(s.shape, 8.0)
    sd = s.double()[..., None]
    y = torch.where(sd > 0, (x / sd).float(), torch.zeros_like(x).float())
    u = (y.round() + z.float()[..., None]).clamp(0, 15)
    return u.to(torch.uint8).view(N, K), s, z.to(torch.uint8)


def values(codes, s, z, group):
    N, K = codes.shape
    return ((codes.view(N, -1, group).double() - z.double()[..., None]) * s.double()[..., None]).view(N, K)


@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(1, 128), (16, 384), (37, 896), (130, 640)])
def test_quantize_pack_unpack(N, K, group, asym):
    g = torch.Generator().manual_seed(N + K + group)
    w = (torch.randn(N, K, generator=g) * 0.05).to(torch.bfloat16)
    w[0, :group] = 0
    w[-1, -group:] = 3e-40                    # bf16 subnormals
    if N > 2:
        w[1, 0], w[1, 1], w[2, 2] = math.inf, -math.inf, math.nan
        w[2, group:] = w[2, group:].abs()     # one-sided groups
    wide = torch.zeros(N, K + 7, dtype=torch.bfloat16)
    wide[:, :K] = w
    codes, s, z = serve.quantize_w4(wide.to(DEV)[:, :K], group, asym)
    rc, rs, rz = ref_quantize(w, group, asym)
    assert torch.equal(s.cpu(), rs) and torch.equal(codes.cpu(), rc)
    assert (z is None) != asym and (z is None or torch.equal(z.cpu(), rz))
    packed = serve.W4Weight.from_codes(codes, s, z)
    assert torch.equal(packed.unpack().cpu(), values(rc, rs, rz, group).to(torch.bfloat16))


def product(M, N, K, group, asym, out=torch.bfloat16, resid=False, pad=0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + M * 7 + N + K)
    codes = torch.randint(0, 16, (N, K), device=DEV, generator=g).to(torch.uint8)
    s = (torch.rand(N, K // group, device=DEV, generator=g) * 0.02).to(torch.bfloat16)
    s[0] = 0
    z = torch.randint(0, 16, s.shape, device=DEV, generator=g).to(torch.uint8) if asym else None
    x = torch.randn(M, K + pad, device=DEV, generator=g).to(torch.bfloat16)[:, :K]
    r = torch.randn(M, N + pad, device=DEV, generator=g).to(torch.bfloat16)[:, :N] if resid else None
    y0 = torch.full((M, N + pad), 5.0, device=DEV, dtype=out)
    y = serve.W4Weight.from_codes(codes, s, z).linear(x, resid=r, out=y0[:, :N])
    w = values(codes, s, torch.full_like(codes[:, :K // group], 8) if z is None else z, group)
    ref = x.double() @ w.t()
    tol = (x.double().abs() @ w.abs().t()) * (8 * 2.0 ** -22 + (K / 32 + 16) * 2.0 ** -23) + 1e-30
    if resid:
        ref = ref + r.double()
        tol = tol + ref.abs() * 2.0 ** -23
    if out == torch.bfloat16:
        tol = tol + 2.0 ** -8 * ref.abs()
    assert ((y.double() - ref).abs() <= tol).all(), ((y.double() - ref).abs() - tol).max()
    assert (y0[:, N:] == 5).all()
    return x, y


@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 2, 8, 9, 16, 17, 31, 32, 33])
def test_rows(M, group, asym):
    product(M, 200, 1152, group, asym, resid=M % 2 == 1)


@pytest.mark.parametrize("N,K,group", [(1, 32, 32), (3, 96, 32), (15, 64, 64), (17, 160, 32), (255, 128, 128),
                                       (896, 4864, 128), (1153, 896, 64), (4099, 2080, 32), (64, 14336, 64)])
@pytest.mark.parametrize("M", [1, 5, 20])
def test_odd_sizes(N, K, group, M):
    product(M, N, K, group, True, out=torch.float32)
    product(M, N, K, group, False)


def test_many_rows_and_strides():
    product(131, 333, 448, 64, True, resid=True, pad=8)
    product(7, 333, 448, 64, False, out=torch.float32, resid=True, pad=24)


def test_no_rows():
    w = serve.W4Weight.quantize(torch.randn(24, 64, device=DEV).to(torch.bfloat16), 32)
    assert w.linear(torch.empty(0, 64, device=DEV, dtype=torch.bfloat16)).shape == (0, 24)


def test_non_finite_inputs_stay_in_their_rows():
    x, y = product(3, 40, 256, 64, False)
    x = x.clone()
    x[1, 5] = math.nan
    x[2, 7] = math.inf
    codes = torch.full((40, 256), 9, device=DEV, dtype=torch.uint8)
    codes[3, 7] = 2
    w = serve.W4Weight.from_codes(codes, torch.ones(40, 4, device=DEV, dtype=torch.bfloat16))
    y = w.linear(x)
    assert torch.isfinite(y[0]).all() and torch.isnan(y[1]).all()
    assert y[2, 3] == -math.inf and (y[2, [i for i in range(40) if i != 3]] == math.inf).all()


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M", [3, 4, 6, 7, 10, 12, 13, 15, 20, 24])
def test_every_number_of_row_tiles(M, out):
    product(M, 2390, 1152, 64, M % 2 == 0, out=out, resid=M % 3 == 0)


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("M", [1, 6, 11, 19, 40])
def test_non_finite_rows_with_many_rows_and_units(M, group):
    """Infinities and NaN in the first and last block of some rows, sums that join over warps, the residual in place."""
    N, K = 1030, 1216 if group == 32 else 1280
    g = torch.Generator(device=DEV).manual_seed(M + group)
    w = serve.W4Weight.quantize((torch.randn(N, K, device=DEV, generator=g) * 0.1).to(torch.bfloat16), group)
    x = torch.randn(M, K, device=DEV, generator=g).to(torch.bfloat16)
    x[0, 3] = math.nan
    if M > 4:
        x[M // 2, K - 1] = -math.inf
    y = torch.randn(M, N, device=DEV, generator=g).to(torch.bfloat16)
    r = y.clone()
    w.linear(x, resid=y, out=y)
    u = w.unpack().double()
    assert torch.isnan(y[0]).all()
    fine = torch.ones(M, dtype=torch.bool, device=DEV)
    fine[0] = False
    if M > 4:
        fine[M // 2] = False
        last = -math.inf * torch.sign(u[:, K - 1])   # NaN where the weight is 0
        assert torch.equal(torch.nan_to_num(y[M // 2].double(), nan=7.0), torch.nan_to_num(last, nan=7.0))
    ref = x.double() @ u.t() + r.double()
    # unpacked weights are rounded to bf16
    tol = (x.double().abs() @ u.abs().t()) * (2.0 ** -9 + 8 * 2.0 ** -22 + (K / 32 + 16) * 2.0 ** -23) + ref.abs() * 2.0 ** -8
    assert ((y.double() - ref).abs() <= tol)[fine].all()


def test_quantized_weight_is_near_the_matrix():
    """Rounding to 4 bits moves a weight by at most half a step (a step's bf16 rounding included)."""
    w = (torch.randn(96, 256, device=DEV) * 0.1).to(torch.bfloat16)
    for asym in (False, True):
        u = serve.W4Weight.quantize(w, 32, asym).unpack()
        g = w.float().view(96, 8, 32)
        step = (g.amax(-1).clamp(min=0) - g.amin(-1).clamp(max=0)) / 15 if asym else g.abs().amax(-1) / 7
        off = (u.float() - w.float()).abs().view(96, 8, 32)
        # the end of the range may lose 7 (15) times the scale's relative rounding of 2^-9
        # (and with zeros, half a step more: the zero is rounded too)
        assert (off <= step[..., None] * (0.5 + 15 * 2.0 ** -9 + (0.5 if asym else 0)) + g.abs() * 2.0 ** -8).all()


def test_side_stream_and_repeats_agree():
    w = serve.W4Weight.quantize((torch.randn(1000, 2048, device=DEV) * 0.1).to(torch.bfloat16), 64)
    x = torch.randn(13, 2048, device=DEV).to(torch.bfloat16)
    a = w.linear(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b = w.linear(x)
    side.synchronize()
    assert torch.equal(a, b)
