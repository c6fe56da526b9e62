"""Windows with first tokens that stay visible (glt_kv8_window_attention) against a 64-bit form; the tolerance is that of
test_gpu_kv8's `attention_ref`, whose kernel this is but for the tokens it goes through."""
import math

import pytest
import torch

from glt_b200 import _lib, serve

pytestmark = pytest.mark.gpu
DEV = "cuda"


def take_error():
    code = _lib.C.c_uint()
    _lib.lib.glt_device_error(_lib.C.byref(code))
    return code.value


class Case:
    """Sequences of which only the blocks that a query of the step may see are in the pool; all else in it is garbage."""

    def __init__(self, fmt, bt, nkv, group, hd, lens, new, window, sinks, seed=0, masked=False):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.fmt, self.bt, self.nkv, self.group, self.hd = fmt, bt, nkv, group, hd
        self.lens, self.new, self.window, self.sinks = lens, new, window, sinks
        seqs, maxb = len(lens), max(-(-(n + new) // bt) for n in lens)
        seen = []
        for n in lens:
            t = torch.arange(n + new)
            see = (t < sinks) | (t > n - window) if window else t >= 0
            seen.append(see)
        nb = sum(len(set((s.nonzero()[:, 0] // bt).tolist())) for s in seen) + 2
        shape = (nb, nkv, bt, hd)
        bad = 0xFF if fmt == "e4m3" else 0
        self.k, self.v = (torch.full(shape, bad, device=DEV, dtype=torch.uint8) for _ in range(2))
        self.ks, self.vs = (torch.full((nb, nkv), math.nan, device=DEV) for _ in range(2))
        self.table = torch.full((seqs, maxb), -1, dtype=torch.int32, device=DEV)
        top, at = 127.0 if fmt == "int8" else 448.0, 0
        for b, s in enumerate(seen):
            for blk in sorted(set((s.nonzero()[:, 0] // bt).tolist())):
                self.table[b, blk] = at
                for pool, scale in ((self.k, self.ks), (self.v, self.vs)):
                    x = torch.randn(nkv, bt, hd, device=DEV, generator=g)
                    sc = x.abs().amax((1, 2)) / top
                    y = x / sc[:, None, None]
                    code = ((y.round() + 128).to(torch.uint8) if fmt == "int8" else y.to(torch.float8_e4m3fn).view(torch.uint8))
                    live = s[blk * bt:(blk + 1) * bt]
                    pool[at, :, :len(live)] = torch.where(live.to(DEV)[None, :, None], code[:, :len(live)], pool[at, :, :len(live)])
                    scale[at] = sc
                at += 1
        self.q = torch.randn(seqs * new, nkv * group, hd, device=DEV, generator=g).to(torch.bfloat16)
        self.mask = None
        if masked:
            self.mask = (torch.rand(seqs, maxb * bt, device=DEV, generator=g) > 0.4).to(torch.uint8)
            self.mask[0] = 0
        self.lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def run(self, **kw):
        cache = serve.Kv8Cache.from_buffers(self.k, self.v, self.ks, self.vs, self.fmt)
        batch = serve.Kv8Batch(self.table, self.lengths, self.q.shape[0], max_new=self.new)
        return cache.attention(batch, self.q, window=self.window, sinks=self.sinks, token_mask=self.mask, **kw)

    def check(self, o, lse):
        val = lambda c: c.double() - 128 if self.fmt == "int8" else c.view(torch.float8_e4m3fn).double()
        scale = 1 / math.sqrt(self.hd)
        for b, past in enumerate(self.lens):
            for i in range(self.new):
                t = torch.arange(past + i + 1, device=DEV)
                if self.window:
                    t = t[(t < self.sinks) | (t > past + i - self.window)]
                if self.mask is not None:
                    t = t[self.mask[b, t] != 0]
                r = b * self.new + i
                got_o, got_l = o[r].double().view(self.nkv, self.group, self.hd), lse[r].double().view(self.nkv, self.group)
                if t.numel() == 0:
                    assert (got_o == 0).all() and (got_l == -math.inf).all()
                    continue
                ids = self.table[b, t // self.bt].long()
                key = (val(self.k[ids, :, t % self.bt]) * self.ks[ids].double()[..., None]).transpose(0, 1)
                v = (val(self.v[ids, :, t % self.bt]) * self.vs[ids].double()[..., None]).transpose(0, 1)
                q = self.q[r].double().view(self.nkv, self.group, self.hd)
                z = torch.einsum("hgd,htd->hgt", q, key) * scale
                want_l = torch.logsumexp(z, -1)
                p = torch.exp(z - want_l[..., None])
                want_o = torch.einsum("hgt,htd->hgd", p, v)
                ds = torch.einsum("hgd,htd->hgt", q.abs(), key.abs()).amax(-1) * scale * (self.hd + 8) * 2.0 ** -23
                tol = 2 * (2.0 ** -11 + 2 * ds)[..., None] * torch.einsum("hgt,htd->hgd", p, v.abs()) + 2.0 ** -8 * want_o.abs() + 1e-30
                assert ((got_o - want_o).abs() <= tol).all(), (b, i)
                assert ((got_l - want_l).abs() <= ds + (4 + t.numel() / 32) * 2.0 ** -23 + 2.0 ** -22 * want_l.abs()).all(), (b, i)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bt,nkv,group,hd", [(16, 2, 7, 64), (32, 1, 4, 128), (64, 2, 3, 64), (128, 1, 8, 128)])
@pytest.mark.parametrize("window,sinks", [(1, 1), (40, 4), (33, 16), (100, 17), (64, 32), (31, 33), (200, 129), (5, 300)])
def test_matches_the_formula(fmt, bt, nkv, group, hd, window, sinks):
    """Windows that touch the first tokens, lie behind them by less than a step, by one, by many; blocks between are gone."""
    lens = [0, 3, sinks, sinks + window - 1, sinks + window, sinks + window + 15, sinks + window + 31, sinks + window + 47, 700, 2011]
    c = Case(fmt, bt, nkv, group, hd, lens, 1, window, sinks, seed=window + sinks)
    take_error()
    c.check(*c.run())
    assert take_error() == 0   # no entry of a block that was given back was looked at


@pytest.mark.parametrize("new,group", [(2, 1), (5, 8), (7, 3)])
@pytest.mark.parametrize("bt", [16, 64])
def test_several_new_tokens(new, group, bt):
    c = Case("e4m3", bt, 2, group, 64, [0, 60, 500, 999, 1003], new, 90, 20, seed=new, masked=True)
    take_error()
    c.check(*c.run())
    assert take_error() == 0


def test_long_streams_in_equal_runs():
    c = Case("int8", 64, 2, 4, 128, [5, 60001, 33, 20000, 9000, 100], 1, 4096, 5, seed=1)
    c.check(*c.run())


def test_all_masked():
    c = Case("int8", 16, 1, 2, 64, [100, 50], 1, 20, 3, seed=2, masked=True)
    c.mask.zero_()
    c.check(*c.run())


@pytest.mark.parametrize("sinks", [10 ** 6, 2 ** 31 - 1, 2 ** 31 - 32])
def test_first_tokens_without_end_are_all(sinks):
    c = Case("int8", 32, 1, 4, 64, [300, 31], 1, 0, 0, seed=3)
    want = c.run()
    c.window, c.sinks = 17, sinks
    got = c.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_without_a_window_or_first_tokens():
    """The same bits as the plain call."""
    c = Case("int8", 32, 2, 4, 64, [300, 31, 0], 2, 0, 0, seed=4)
    want = c.run()
    c.sinks = 9
    got = c.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    c = Case("e4m3", 64, 1, 4, 128, [300, 31, 900], 1, 100, 7, seed=5)
    c.sinks = 0
    want = c.run()
    cache = serve.Kv8Cache.from_buffers(c.k, c.v, c.ks, c.vs, c.fmt)
    got = cache.attention(serve.Kv8Batch(c.table, c.lengths, 3), c.q, window=100)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_graph_follows_the_lengths():
    c = Case("int8", 16, 2, 4, 64, [1500, 1300], 1, 0, 0, seed=6)   # all blocks there
    c.window, c.sinks = 200, 6
    c.run()
    cache = serve.Kv8Cache.from_buffers(c.k, c.v, c.ks, c.vs, c.fmt)
    batch = serve.Kv8Batch(c.table, c.lengths, 2)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, lse = cache.attention(batch, c.q, window=200, sinks=6)
    for lens in ([1500, 1300], [0, 5], [210, 190], [700, 0]):
        c.lens = lens
        c.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        c.check(o, lse)
