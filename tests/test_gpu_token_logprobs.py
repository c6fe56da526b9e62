"""Token log probabilities, entropy, alternatives and gradient
(glt_token_logprobs, glt_token_logprobs_bwd) against 64-bit forms and
differences.

Tolerances: a row's sums are positive and run in 32 bits, at most V/64 + 64
additions deep, over terms whose exponent z - max carries 2^-23 |z|; so a
relative error e = (V/64 + 64) 2^-24 + 4 * 2^-23 max|z| + 2^-21 in each sum."""
import math

import pytest
import torch

from glt_b200 import _lib, serve

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reference(x, t, scale, top):
    x = x.double()
    z = x * scale
    lse = torch.logsumexp(z, -1)
    lq = z - lse[:, None]
    p = lq.exp()
    ent = -torch.where(p > 0, p * lq, torch.zeros_like(p)).sum(-1)
    lp = torch.where(t < 0, torch.zeros_like(lse), lq.gather(1, t.clamp(min=0).long()[:, None])[:, 0])
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    return lp, ent, lse, ids, lq.gather(1, ids), p, lq


def eps(x, scale):
    fin = x.double()[torch.isfinite(x.double())]
    big = float(fin.abs().max()) * scale if fin.numel() else 0.0
    return (x.shape[1] / 64 + 64) * 2.0 ** -24 + 4 * 2.0 ** -23 * big + 2.0 ** -21, big


def compare(x, t, scale, top, train=True, in_place=False):
    f = serve.token_logprobs(x, t, scale=scale, top=top)
    lp, ent, lse, ids, tlp, p, lq = reference(x, t, scale, top)
    e, big = eps(x, scale)
    tol_l = e + 2.0 ** -22 * big
    assert ((f.lse.double() - lse).abs() <= tol_l).all()
    ok = torch.isfinite(lp)
    assert torch.equal(f.logp.double()[~ok], lp[~ok])
    assert ((f.logp.double() - lp).abs()[ok] <= 2 * tol_l).all()
    tol_h = (2 * e + 2.0 ** -21) * (1 + ent) + 2.0 ** -21 * big
    assert ((f.entropy.double() - ent).abs() <= tol_h).all(), (f.entropy.double() - ent).abs().max()
    if top:
        assert torch.equal(f.top_ids.long(), ids)
        fin = torch.isfinite(tlp)
        assert torch.equal(f.top_logp.double()[~fin], tlp[~fin])
        assert ((f.top_logp.double() - tlp).abs()[fin] <= 2 * tol_l).all()
    if not train:
        return
    g = torch.Generator(device=DEV).manual_seed(x.shape[1])
    dl, de = torch.randn(2, x.shape[0], device=DEV, generator=g)
    for a, b in ((dl, de), (dl, None), (None, de)):
        src = x.clone() if in_place else x
        d = serve.token_logprobs_bwd(src, t, f, a, b, out=src if in_place else None)
        da = torch.zeros_like(dl).double() if a is None else torch.where(t < 0, torch.zeros_like(a), a).double()
        db = torch.zeros_like(de).double() if b is None else b.double()
        hot = torch.zeros_like(p).scatter_(1, t.clamp(min=0).long()[:, None], 1.0)
        spread = torch.where(p > 0, lq + ent[:, None], torch.zeros_like(p))
        want = scale * (da[:, None] * (hot - p) - db[:, None] * p * spread)
        tol = scale * p * (da.abs()[:, None] * 3 * tol_l + db.abs()[:, None] *
                           (3 * tol_l * spread.abs() + 2 * tol_l + tol_h[:, None])) + 2.0 ** -22 * want.abs() + 1e-37
        tol = tol + scale * hot * da.abs()[:, None] * 2.0 ** -22
        if x.dtype == torch.bfloat16:
            tol = tol + 2.0 ** -8 * want.abs()
        assert ((d.double() - want).abs() <= tol).all(), ((d.double() - want).abs() - tol).max()


def rows(R, V, dtype, seed, sigma=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(R, V, device=DEV, generator=g) * sigma).to(dtype)
    t = torch.randint(0, V, (R,), device=DEV, generator=g).to(torch.int32)
    t[::5] = -1
    return x, t


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,V,top", [(1, 1, 1), (3, 2, 2), (2, 7, 7), (5, 31, 5), (4, 32, 32), (3, 33, 32), (2, 255, 20),
                                     (7, 257, 1), (2, 1000, 32), (3, 4099, 8), (1, 32003, 20), (2, 151936, 32),
                                     (300, 515, 4), (1200, 1025, 0), (900, 20001, 3)])
def test_sizes(R, V, top, dtype):
    x, t = rows(R, V, dtype, R + V)
    compare(x, t, 1.0, top)
    compare(x, t, 0.6, min(top, 3), in_place=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("off,pad", [(0, 3), (1, 0), (3, 5), (5, 8)])
def test_strides_and_alignment(dtype, off, pad):
    """Rows that start anywhere an element may."""
    R, V = 4, 5003
    x, t = rows(R, V, dtype, 3)
    wide = torch.zeros(R * (V + pad) + off + 8, device=DEV, dtype=dtype)
    view = wide[off:off + R * (V + pad)].view(R, V + pad)[:, :V]
    view.copy_(x)
    compare(view, t, 1.3, 6)
    f = serve.token_logprobs(view, t, top=0)
    out = torch.full((R * (V + 2) + 9,), 3.0, device=DEV, dtype=dtype)
    o = out[1:1 + R * (V + 2)].view(R, V + 2)[:, :V]
    serve.token_logprobs_bwd(view, t, f, f.lse, f.entropy, out=o)
    assert torch.equal(o, serve.token_logprobs_bwd(x, t, f, f.lse, f.entropy))
    assert (out[0] == 3) and (out[1 + R * (V + 2):] == 3).all()
    assert (out[1:1 + R * (V + 2)].view(R, V + 2)[:, V:] == 3).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ties_take_the_lowest_index(dtype):
    V = 20000
    g = torch.Generator(device=DEV).manual_seed(1)
    few = torch.randint(-2, 3, (3, V), device=DEV, generator=g).to(dtype)   # thousands of equal maxima
    flat = torch.zeros(2, V, device=DEV, dtype=dtype)
    flat[1, 1::2] = -0.0                                                    # -0 equals +0
    falling = torch.arange(V, 0, -1, device=DEV).to(dtype)[None] / 1024    # the largest ones side by side
    rising = falling.flip(1)
    comb = torch.zeros(1, V, device=DEV, dtype=dtype)
    comb[0, 5::2048] = 1.0                                                  # all in one thread's share
    comb[0, 4::512] = 0.5
    x = torch.cat((few, flat, falling, rising, comb))
    t = torch.zeros(x.shape[0], device=DEV, dtype=torch.int32)
    compare(x, t, 1.0, 32, train=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_forbidden_tokens_and_empty_rows(dtype):
    x, t = rows(5, 3001, dtype, 2)
    x[0, 7:] = -math.inf                     # fewer allowed tokens than alternatives asked for
    x[1] = -math.inf                         # nothing allowed
    x[2, t[2].long()] = -math.inf            # the given token is forbidden
    x[3] = torch.finfo(dtype).min            # the lowest finite value everywhere
    x[3, 9] = 0
    t[2] = 77
    x[2, 77] = -math.inf
    t[1] = 4
    keep = torch.tensor([0, 2, 3, 4], device=DEV)
    compare(x[keep].contiguous(), t[keep].contiguous(), 1.0, 20)
    f = serve.token_logprobs(x, t, top=20)
    assert f.lse[1] == -math.inf and f.logp[1] == -math.inf and f.entropy[1] == 0
    assert torch.equal(f.top_ids[1], torch.arange(20, device=DEV, dtype=torch.int32)) and (f.top_logp[1] == -math.inf).all()
    d = serve.token_logprobs_bwd(x, t, f, torch.ones(5, device=DEV), torch.ones(5, device=DEV))
    assert (d[1] == 0).all() and torch.isfinite(d.float()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nan_and_infinity_give_nan_in_their_row_only(dtype):
    x, t = rows(4, 2049, dtype, 4)
    t[:] = 3
    x[0, 100], x[1, 2048], x[1, 5] = math.nan, math.inf, math.nan
    x[2, :] = math.nan
    f = serve.token_logprobs(x, t, top=5)
    for s in (f.lse, f.logp, f.entropy):
        assert torch.isnan(s[:3]).all() and torch.isfinite(s[3])
    assert torch.isnan(f.top_logp[:3]).all() and f.top_ids[1, 0] == 2048
    clean = x[0].float().clone()
    clean[100] = -math.inf
    assert torch.equal(f.top_ids[0].long(), torch.sort(clean, descending=True, stable=True).indices[:5])
    assert torch.equal(f.top_ids[2], torch.arange(5, device=DEV, dtype=torch.int32))
    d = serve.token_logprobs_bwd(x, t, f, torch.ones(4, device=DEV))
    assert torch.isnan(d[:3]).all() and torch.isfinite(d[3]).all()


def test_gradient_against_differences():
    """Central differences of the 64-bit forward (step 1e-5: error of order 1e-9)."""
    x, t = rows(3, 41, torch.float32, 6, sigma=1.5)
    dl, de = torch.randn(2, 3, device=DEV)
    f = serve.token_logprobs(x, t, scale=1.4)
    d = serve.token_logprobs_bwd(x, t, f, dl, de)

    def loss(y):
        lp, ent = reference(y, t, 1.4, 1)[:2]
        return (lp * dl.double() + ent * de.double()).sum()

    for r in range(3):
        for v in range(41):
            h = torch.zeros(3, 41, device=DEV, dtype=torch.float64)
            h[r, v] = 1e-5
            diff = (loss(x.double() + h) - loss(x.double() - h)) / 2e-5
            assert abs(float(diff) - float(d[r, v])) <= 2e-6 * (1 + abs(float(diff)))


def test_without_targets_and_out_of_range_targets():
    x, _ = rows(3, 515, torch.bfloat16, 7)
    f = serve.token_logprobs(x, None, top=2)
    assert f.logp is None
    code = _lib.C.c_uint()
    _lib.lib.glt_device_error(_lib.C.byref(code))
    t = torch.tensor([515, 2, 10 ** 9], device=DEV, dtype=torch.int32)
    g = serve.token_logprobs(x, t)
    _lib.lib.glt_device_error(_lib.C.byref(code))
    assert code.value == 2 and g.logp[0] == 0 and g.logp[2] == 0 and g.logp[1] < 0
    assert torch.equal(f.lse, g.lse)
    d = serve.token_logprobs_bwd(x, t, g, torch.ones(3, device=DEV))
    assert (d[0] == 0).all() and (d[2] == 0).all() and (d[1] != 0).any()


def test_offsets_past_32_bits():
    R, V = 3, 1 << 20
    ld = (1 << 31) + 8                      # rows 4 GiB apart
    buf = torch.empty(2 * ld + V, device=DEV, dtype=torch.bfloat16)
    view = torch.as_strided(buf, (R, V), (ld, 1))
    x, t = rows(R, V, torch.bfloat16, 8)
    view.copy_(x)
    a, b = serve.token_logprobs(view, t, top=4), serve.token_logprobs(x, t, top=4)
    assert torch.equal(a.lse, b.lse) and torch.equal(a.top_ids, b.top_ids)
    d = serve.token_logprobs_bwd(view, t, a, a.lse, out=view)
    assert torch.equal(d, serve.token_logprobs_bwd(x, t, b, b.lse))
    del buf, view, d
    torch.cuda.empty_cache()


def test_equal_maxima_in_the_last_vectors_cost_no_second_pass():
    """Threads whose maxima are equal and lie in the row's last, short batch of vectors keep
    different bounds (rows of this kind took twenty times as long as others)."""
    V, R = 128256, 64
    x = torch.full((R, V), -8.0, device=DEV, dtype=torch.bfloat16)
    x += torch.randn(R, V, device=DEV).to(torch.bfloat16)
    x[:, -2000::8] = 9.0          # one element in each of the last 250 vectors
    x[:, :3] = 20.0
    t = torch.zeros(R, device=DEV, dtype=torch.int32)
    compare(x, t, 1.0, 5, train=False)
    plain = x.clone()
    plain[:, -2000::8] = torch.arange(250, device=DEV).to(torch.bfloat16) / 100

    def took(y):
        serve.token_logprobs(y, t, top=5)
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(20):
            serve.token_logprobs(y, t, top=5)
        b.record()
        b.synchronize()
        return a.elapsed_time(b)

    assert min(took(x) for _ in range(3)) < 4 * min(took(plain) for _ in range(3))
