"""Rounding to 4 bits at the ends of bf16's range (glt_w4_quantize with zeros): the scale is the range over 15 also where
the range itself, from -3.4e38 to 3.4e38, is beyond a float, and no weight of a finite matrix becomes NaN."""
import pytest
import torch

from glt_b200 import serve

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("lo,hi", [(-1.0, 1.0), (-1.0, 0.25), (-0.3, 1.0), (-0.7, 0.6), (0.0, 1.0), (-1.0, 0.0)])
def test_ranges_up_to_the_largest_numbers(lo, hi, group):
    top = torch.finfo(torch.bfloat16).max
    g = torch.Generator(device=DEV).manual_seed(group)
    w = (torch.rand(24, 256, device=DEV, generator=g).double() * (hi - lo) + lo) * top
    w[:, 0::group], w[:, 1::group] = lo * top, hi * top
    w = w.to(torch.bfloat16)
    codes, s, z = serve.quantize_w4(w, group, asym=True)
    x = w.double().view(24, -1, group)
    want = ((x.amax(-1).clamp(min=0) - x.amin(-1).clamp(max=0)) / 15)
    assert ((s.double() - want).abs() <= 2.0 ** -8 * want).all()          # one rounding to bf16 (and one to 32 bits)
    assert ((z.double() - (-x.amin(-1).clamp(max=0) / s.double())).abs() <= 0.5 + 1e-6).all()
    back = (codes.view(24, -1, group).double() - z.double()[..., None]) * s.double()[..., None]
    # half a step for the value, half for the zero, the ends of the range with their scale's rounding
    assert ((back - x).abs() <= s.double()[..., None] * (1 + 15 * 2.0 ** -8)).all()
    y = serve.W4Weight.from_codes(codes, s, z).linear(torch.full((2, 256), 2.0 ** -8, device=DEV).to(torch.bfloat16),
                                                      out_dtype=torch.float32)
    ref = back.sum((1, 2)) * 2.0 ** -8
    assert torch.isfinite(y).all() and ((y.double() - ref).abs() <= 2.0 ** -14 * back.abs().sum((1, 2)) * 2.0 ** -8).all()
