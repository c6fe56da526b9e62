"""Token log probabilities of logits far from 0 (glt_token_logprobs) against 64-bit forms.

A row's statistics are taken relative to its maximum, so their error does not grow with it: with d = scale (x - max),
a term exp(d) is off by 2^-21 and 2^-22 |d| of itself (|d| exp(d) <= 1), and sums of V terms run at most V + 16
additions deep for V <= 64, V / 64 + 64 for more.  So ls = log sum exp d is off by e below, logp by e + 2^-22 |d|,
the entropy by 2 e (1 + entropy); only lse = scale max + ls carries the maximum's own 2^-23."""
import math

import pytest
import torch

from glt_b200 import serve

pytestmark = pytest.mark.gpu
DEV = "cuda"


def compare(x, scale, top=0):
    R, V = x.shape
    d64 = (x.double() - x.double().amax(-1, keepdim=True)) * scale
    ls = torch.logsumexp(d64, -1)
    lq = d64 - ls[:, None]
    p = lq.exp()
    ent = -torch.where(p > 0, p * lq, torch.zeros_like(p)).sum(-1)
    lse = x.double().amax(-1) * scale + ls
    e = (V + 16 if V <= 64 else V / 64 + 64) * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -22
    pick = list(range(min(V, 5))) + [V // 2, V - 1] + [int(x[0].float().argmax())]
    for v in sorted(set(pick)):
        t = torch.full((R,), v, device=DEV, dtype=torch.int32)
        f = serve.token_logprobs(x, t, scale=scale, top=top)
        want = lq[:, v]
        got = f.logp.double()
        huge = want < -3.3e38                      # beyond fp32
        assert (got[huge] < -3e38).all()
        assert ((got - want).abs() <= e + 2.0 ** -22 * d64[:, v].abs())[~huge].all(), ((got - want).abs()[~huge].max(), e)
        assert (got <= 0).all()
    far = lse.abs() > torch.finfo(torch.float32).max * (1 + 2.0 ** -24)
    assert ((f.lse.double() - lse).abs() <= 2.0 ** -23 * lse.abs() + e)[~far].all() and torch.isinf(f.lse[far]).all()
    assert ((f.entropy.double() - ent).abs() <= 2 * e * (1 + ent)).all(), (f.entropy.double() - ent).abs().max()
    if top:
        ids = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(f.top_ids.long(), ids)
        want = lq.gather(1, ids)
        ok = want > -3.3e38
        assert ((f.top_logp.double() - want).abs() <= e + 2.0 ** -22 * d64.gather(1, ids).abs())[ok].all()


def spread(R, V, at, step, dtype, seed):
    """Rows whose maximum is `at`, the others a few multiples of `step` (a multiple of at's spacing) below."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = at - torch.randint(0, 40, (R, V), device=DEV, generator=g).double() * step
    x[:, V // 3] = at
    y = x.to(dtype)
    assert torch.equal(y.double(), x)
    return y


@pytest.mark.parametrize("scale", [1.0, 0.37, 3.0])
@pytest.mark.parametrize("V", [9, 64, 1000, 20001])
@pytest.mark.parametrize("at,step", [(float(2 ** 20 + 3), 0.125), (float(2 ** 21 + 1), 0.25), (float(2 ** 23 - 1), 0.5),
                                     (-float(2 ** 22 - 1), 0.5), (float(2 ** 31), 256.0), (2.0 ** 60, 2.0 ** 37)])
def test_large_maxima_keep_their_differences(at, step, V, scale):
    compare(spread(3, V, at, step, torch.float32, V), scale, top=min(V, 5))


@pytest.mark.parametrize("scale", [1.0, 0.25, 3.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [8, 1001, 20000])
def test_logits_at_the_type_s_ends(V, dtype, scale):
    top, low = torch.finfo(dtype).max, torch.finfo(dtype).min
    g = torch.Generator(device=DEV).manual_seed(V)
    x = torch.empty(6, V, device=DEV, dtype=dtype)
    x[0] = top                                         # all equal
    x[1] = low
    x[1, V // 2] = top                                 # one token
    x[2] = torch.where(torch.rand(V, device=DEV, generator=g) < 0.5, top, low).to(dtype)
    x[3] = torch.randn(V, device=DEV, generator=g).to(dtype)
    x[3, 1] = top
    x[4] = low
    x[5] = (torch.rand(V, device=DEV, generator=g) * 2 - 1).to(dtype) * (top / 2)
    x[2, 0] = top
    compare(x, scale, top=4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("at", [20.3, 37.7, 61.1, 1003.0, 3.3e4, 7.1e5])
def test_one_likely_token_has_probability_one(at, dtype):
    """log p of the only token is 0, and no log probability is above it."""
    g = torch.Generator(device=DEV).manual_seed(int(at))
    for V in (8, 515, 20001):
        x = torch.full((16, V), -math.inf, device=DEV, dtype=dtype)
        m = (at * (1 + torch.rand(16, device=DEV, generator=g) / 2)).to(dtype)
        x[:, V // 2] = m
        x[8:] = torch.maximum(x[8:], (m[8:, None] - 200 - at / 2).to(dtype))   # too far below to count
        t = torch.full((16,), V // 2, device=DEV, dtype=torch.int32)
        for scale in (1.0, 0.7, 1.9):
            f = serve.token_logprobs(x, t, scale=scale)
            assert (f.logp == 0).all() and (f.entropy.abs() <= 2.0 ** -21).all()
            want = m.double() * scale
            assert ((f.lse.double() - want).abs() <= 2.0 ** -23 * want).all()


@pytest.mark.parametrize("at,step", [(24.0, 0.125), (60.5, 0.25), (1000.0, 0.5), (32768.0, 0.25), (524288.0, 0.25)])
@pytest.mark.parametrize("V", [8, 33, 1000, 20001])
def test_confident_rows_keep_their_digits(at, step, V):
    for seed in range(4):
        compare(spread(5, V, at + seed * step, step, torch.float32, seed), 1.0 if seed % 2 else 0.77)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [0.5, 1.0, 3.0])
def test_forbidden_tokens_below_a_very_low_maximum(dtype, scale):
    """A logit of -inf has log probability -inf also where the maximum times the scale is beyond the float range."""
    low = torch.finfo(dtype).min
    x = torch.full((2, 700), -math.inf, device=DEV, dtype=dtype)
    x[:, 5], x[1, 600] = low, low
    for v, want in ((5, [0.0, -math.log(2)]), (3, [-math.inf] * 2), (600, [-math.inf, -math.log(2)])):
        f = serve.token_logprobs(x, torch.full((2,), v, device=DEV, dtype=torch.int32), scale=scale, top=3)
        want = torch.tensor(want, device=DEV)
        assert torch.equal(torch.isinf(f.logp), torch.isinf(want)) and not torch.isnan(f.logp).any()
        fin = torch.isfinite(want)
        assert ((f.logp - want).abs()[fin] <= 2.0 ** -20).all()
        assert (f.top_logp[0, 1:] == -math.inf).all() and (f.top_logp[1, 2] == -math.inf)
