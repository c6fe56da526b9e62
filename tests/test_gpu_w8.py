"""Products in 8-bit integers (glt_w8_*, serve.W8Weight) against plain 64-bit forms.

Quantising without a norm is held to equality: a scale is the 32-bit quotient of a maximum, a code the nearest to a
32-bit quotient.  Sums of products of codes are exact integers, so that a product's error is that of
its roundings: the integer to 24 bits, two products, the residual's sum (four times 2^-24 of the magnitudes involved), and
bf16's 2^-8 / 2 (`finfo.eps / 2`) of the result where that is its type."""
import math

import pytest
import torch

from glt_b200 import _lib, serve

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def codes_ref(y):
    """(codes, scales) of values given in 32 bits, by the rule in 64."""
    finite = torch.isfinite(y).all(1)
    peak = torch.where(finite, y.double().abs().amax(1), torch.zeros(1, device=DEV, dtype=torch.float64))
    s = (peak / 127).float()
    quot = (y.double() / s.double()[:, None]).float()
    c = torch.where((s > 0)[:, None] & finite[:, None], quot.round().clamp(-127, 127), torch.zeros_like(quot))
    return c.to(torch.int8), torch.where(finite, s, torch.full_like(s, math.nan))


def product_ref(c, s, wc, ws, resid=None):
    """(y, tolerance before the result's own rounding) in 64 bits."""
    y = (c.double() @ wc.double().t()) * ws.double() * s.double()[:, None]
    tol = 3 * 2.0 ** -24 * y.abs()
    if resid is not None:
        tol = tol + 2.0 ** -24 * (y.abs() + resid.double().abs())
        y = y + resid.double()
    return y, tol + 1e-37


def near(got, want, tol):
    if got.dtype == torch.bfloat16:
        tol = tol + torch.finfo(torch.bfloat16).eps / 2 * (want.abs() + tol)
    assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() - tol).max()


def weight(N, K, seed, spread=True):
    g = gen(seed)
    codes = torch.randint(-127, 128, (N, K), device=DEV, generator=g, dtype=torch.int8)
    return codes, torch.rand(N, device=DEV, generator=g) * 0.01 + (1e-4 if spread else 0.01)


@pytest.mark.parametrize("rows,K", [(1, 1), (3, 7), (2, 15), (5, 16), (4, 17), (300, 100), (9, 2048), (2, 4096), (3, 4097), (1300, 4096),
                                    (6, 8192), (5, 9001), (3, 16384), (2, 20000), (1, 131071)])
def test_codes_are_the_rule(rows, K):
    x = (torch.randn(rows, K, device=DEV, generator=gen(K)) * torch.exp(3 * torch.randn(rows, 1, device=DEV, generator=gen(1)))).to(torch.bfloat16)
    q = serve.quantize_rows(x)
    c, s = codes_ref(x.float())
    assert torch.equal(q.scales, s) and torch.equal(q.codes, c)
    padded = torch.as_strided(q.codes, (rows, (K + 15) // 16 * 16), q.codes.stride())
    assert (padded[:, K:] == 0).all()


def test_codes_at_every_boundary():
    """Quotients on and next to k + 1/2, where one more rounding would choose the other code."""
    tops = torch.tensor([127.0, 1.0, 3.0, 100.5, 255.0, 0.0078125, 1e-30, 3e38, 1.5e-38, 2e-40], device=DEV).to(torch.bfloat16)
    half = (torch.arange(-127, 127, device=DEV).double() + 0.5)
    rows = []
    for t in tops:
        y = (half * (t.double() / 127)).to(torch.bfloat16)
        bits = y.view(torch.int16)
        rows.append(torch.cat((t[None], -t[None], y, (bits + 1).view(torch.bfloat16), (bits - 1).view(torch.bfloat16))))
    x = torch.stack(rows)
    x = torch.where(x.float().abs() <= tops[:, None].float(), x, torch.zeros_like(x))
    q = serve.quantize_rows(x)
    c, s = codes_ref(x.float())
    assert torch.equal(q.scales, s) and torch.equal(q.codes, c)


@pytest.mark.parametrize("K", [300, 4096, 5000, 20001])
def test_rows_without_a_scale(K):
    """Zeros give zeros, whatever holds an infinity or NaN gives NaN, and other rows do not see it."""
    x = torch.randn(7, K, device=DEV, generator=gen(5)).to(torch.bfloat16)
    x[1] = 0
    x[2, K - 1], x[3, 0], x[4, K // 2] = math.inf, -math.inf, math.nan
    x[5] = -0.0
    q = serve.quantize_rows(x)
    c, s = codes_ref(x.float())
    assert torch.equal(q.codes, c) and torch.equal(torch.isnan(q.scales), torch.isnan(s))
    assert torch.equal(q.scales[[0, 1, 5, 6]], s[[0, 1, 5, 6]]) and q.scales[1] == 0
    codes, scales = weight(70, K, 6)
    y = serve.W8Weight.from_codes(codes, scales).linear(x)
    assert torch.isnan(y[2:5]).all() and (y[[1, 5]] == 0).all() and torch.isfinite(y[[0, 6]]).all()


@pytest.mark.parametrize("rows,K,amp", [(3, 1000, 1.0), (1500, 896, 4.0), (2, 4096, 1e25), (2, 4096, 1e-25), (4, 14336, 1.0), (2, 20000, 2.0),
                                        (2, 20000, 1e25)])
def test_codes_of_a_norm(rows, K, amp):
    """The norm is in 32 bits: its sum of K squares is off by at most (K / threads + 16) 2^-24, taken as 64 of them, so a value is
    off by some 70 * 2^-24, and a quotient of up to 127 by 127 * 140 * 2^-24: only quotients as near as that to k + 1/2
    may have the other code."""
    g = gen(K)
    x = (torch.randn(rows, K, device=DEV, generator=g) * amp).to(torch.bfloat16)
    w = (1 + 0.3 * torch.randn(K, device=DEV, generator=g)).to(torch.bfloat16)
    eps = 1e-6
    q = serve.quantize_rows(x, w, eps)
    y = x.double() / torch.sqrt(x.double().square().mean(1, keepdim=True) + eps) * w.double()
    s = y.abs().amax(1) / 127
    off = 70 * 2.0 ** -24
    assert ((q.scales.double() - s).abs() <= 2 * off * s).all()
    quot = torch.where(s[:, None] > 0, y / s[:, None], torch.zeros_like(y))
    assert ((q.codes.double() - quot).abs() <= 0.5 + 127 * 2 * off + 1e-4 * (amp < 1e-20)).all()


SIZES = [(1, 1, 1), (1, 128, 128), (2, 127, 129), (8, 300, 1000), (16, 129, 640), (17, 896, 4864), (33, 1000, 97), (64, 2100, 4096),
         (65, 640, 2048), (130, 4096, 1024), (200, 6144, 300), (300, 37900, 130), (577, 257, 513), (2047, 896, 384), (1, 19, 131071)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("out,resid", [(torch.bfloat16, False), (torch.float32, True), (torch.bfloat16, True)])
def test_linear(M, N, K, out, resid):
    g = gen(M + N + K)
    x = (torch.randn(M, K, device=DEV, generator=g) * torch.exp(torch.randn(M, 1, device=DEV, generator=g))).to(torch.bfloat16)
    codes, scales = weight(N, K, 1)
    w = serve.W8Weight.from_codes(codes, scales)
    r = torch.randn(M, N, device=DEV, generator=g).to(torch.bfloat16) if resid else None
    y = w.linear(x, resid=r, out_dtype=out)
    c, s = codes_ref(x.float())
    want, tol = product_ref(c, s, codes, scales, r)
    assert y.dtype == out and y.shape == (M, N)
    near(y, want, tol)
    assert torch.equal(y, w.linear_rows(serve.quantize_rows(x), resid=r, out_dtype=out))
    # sums of integers do not depend on their order
    assert torch.equal(y, w.linear(x, resid=r, out_dtype=out))


def test_the_largest_sums_do_not_overflow():
    """131071 products of -128 by -128 are 64 short of 2^31 thousands: the last size that fits."""
    K = 131071
    codes = torch.full((3, K), -128, device=DEV, dtype=torch.int8)
    w = serve.W8Weight.from_codes(codes, torch.ones(3, device=DEV))
    rows = serve.quantize_rows(torch.zeros(2, K, device=DEV, dtype=torch.bfloat16))
    rows.codes.fill_(-128)
    rows.scales.fill_(1.0)
    assert (w.linear_rows(rows, out_dtype=torch.float32) == float(K * 128 * 128)).all()


@pytest.mark.parametrize("M,N,K", [(5, 200, 500), (70, 333, 1024), (700, 300, 384)])
def test_strides_and_places(M, N, K):
    """Rows of x, out and resid that lie apart, unaligned addresses, and a result over its residual."""
    g = gen(9)
    codes, scales = weight(N, K, 2)
    w = serve.W8Weight.from_codes(codes, scales)
    x = torch.randn(M, K + 11, device=DEV, generator=g).to(torch.bfloat16)[:, 3:3 + K]
    r = torch.randn(M, N + 5, device=DEV, generator=g).to(torch.bfloat16)[:, 1:1 + N]
    want = w.linear(x.contiguous(), resid=r.contiguous())
    held = torch.full((M, N + 7), 9.0, device=DEV, dtype=torch.bfloat16)
    out = held[:, 2:2 + N]
    assert w.linear(x, resid=r, out=out) is out
    assert torch.equal(out, want) and (held[:, :2] == 9).all() and (held[:, 2 + N:] == 9).all()
    w.linear(x, resid=r, out=r)
    assert torch.equal(r, want)
    norm = torch.rand(K + 1, device=DEV, generator=g).to(torch.bfloat16)[1:]
    a, b = w.linear(x, norm=norm.clone()), w.linear(x.contiguous(), norm=norm)
    assert torch.equal(a, b)


def test_weights_by_rows_and_from_codes():
    g = gen(3)
    m = (torch.randn(130, 999, device=DEV, generator=g) * 0.02).to(torch.bfloat16)
    a = serve.W8Weight.quantize(m)
    c, s = codes_ref(m.float())
    b = serve.W8Weight.from_codes(c, s)
    x = torch.randn(9, 999, device=DEV, generator=g).to(torch.bfloat16)
    assert torch.equal(a.codes, c) and torch.equal(a.linear(x), b.linear(x))
    assert torch.equal(a.linear(x), serve.W8Weight.from_codes(c.t().contiguous().t(), s).linear(x))


def test_no_rows():
    w = serve.W8Weight.from_codes(*weight(40, 100, 1))
    x = torch.empty(0, 100, device=DEV, dtype=torch.bfloat16)
    assert w.linear(x).shape == (0, 40) and w.linear_rows(serve.quantize_rows(x)).shape == (0, 40)


def test_graphs_and_streams():
    """Two captured calls replay side by side with new inputs, and a call runs on the current stream."""
    w = serve.W8Weight.from_codes(*weight(3000, 2000, 4))
    xs = [torch.randn(12, 2000, device=DEV, generator=gen(i)).to(torch.bfloat16) for i in range(2)]
    w.linear(xs[0])
    side = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for x, st in zip(xs, side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(w.linear(x))
        graphs.append(g)
    for turn in range(20):
        for i, x in enumerate(xs):
            x.copy_(torch.randn(12, 2000, device=DEV, generator=gen(10 + 2 * turn + i)))
        want = [w.linear(x) for x in xs]
        torch.cuda.synchronize()
        for g, st in zip(graphs, side):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    with torch.cuda.stream(side[0]):
        y = w.linear(xs[0])
    torch.cuda.synchronize()
    assert torch.equal(y, want[0])


def test_no_error_is_left():
    code = _lib.C.c_uint()
    assert _lib.lib.glt_device_error(_lib.C.byref(code)) == 0 and code.value == 0
