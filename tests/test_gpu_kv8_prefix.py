"""Attention of a batch behind a shared prefix (glt_kv8_prefix_attention) against a 64-bit form.

Tolerance, for scores s (base 2) and weights p of the exact softmax:
  * a score is hd products and two scales in 32 bits, tensor cores truncate: |ds| <= (hd + 8) 2^-23 max sum|q||k| scale;
  * the exponent s + log2(scale of v) - reference is rounded: (|s| + 150) 2^-23 more, in units of ln 2;
  * a weight is rounded to f16, 2^-11, and below f16's normal range by at most half of 2^-24, where the reference, which
    the row's largest summand reaches, counts 2^10: 2^-35 of that summand a token, times the largest code (512);
  * values whose scale is below 2^-90 count as 0: what they add, sum p |v| over those, is missing;
  * the result to bf16, eps / 2."""
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


def values(codes, fmt):
    return codes.double() - 128 if fmt == "int8" else codes.view(torch.float8_e4m3fn).double()


class Case:
    """A cache of random codes and scales; sequences of given lengths behind a prefix; garbage wherever nothing lies."""

    def __init__(self, fmt, bt, nkv, group, hd, pre, own, news, seed=0, q_amp=1.0, room=0, spread=0.0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.fmt, self.bt, self.nkv, self.group, self.hd, self.pre, self.own, self.news = fmt, bt, nkv, group, hd, pre, own, news
        self.nh, seqs = nkv * group, len(own)
        pre_blocks = -(-pre // bt) + room
        maxb = max(1, max(-(-(a + b) // bt) for a, b in zip(own, news)))
        nb = pre_blocks + seqs * maxb + 3
        shape = (nb, nkv, bt, hd)
        if fmt == "int8":
            self.k, self.v = (torch.randint(1, 256, shape, device=DEV, generator=g).to(torch.uint8) for _ in range(2))
        else:
            self.k, self.v = ((torch.randn(shape, device=DEV, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
                              for _ in range(2))
        top = 127.0 if fmt == "int8" else 448.0
        self.ks, self.vs = ((torch.rand(nb, nkv, device=DEV, generator=g) + 0.5) * 3 / top *
                            torch.exp2(torch.randn(nb, nkv, device=DEV, generator=g) * s) for s in (0.0, spread))
        perm = torch.randperm(nb, generator=torch.Generator().manual_seed(seed + 1)).to(torch.int32)
        self.blocks = perm[:pre_blocks].to(DEV)
        self.table = perm[pre_blocks:pre_blocks + seqs * maxb].view(seqs, maxb).to(DEV).contiguous()
        rows = sum(news)
        W = (self.nh + 2 * nkv) * hd
        self.q = (torch.randn(rows, W, device=DEV, generator=g) * q_amp).to(torch.bfloat16)[:, :self.nh * hd].unflatten(1, (self.nh, hd))
        self.scale, self.mask = 1 / math.sqrt(hd), None
        self.length = torch.tensor([pre], dtype=torch.int32, device=DEV)
        self.lengths = torch.tensor(own, dtype=torch.int32, device=DEV)
        # what no query sees: the rest of the last blocks, and whole ones behind
        bad = 0xFF if fmt == "e4m3" else 0
        for b in range(pre // bt, pre_blocks):
            i, lo = int(self.blocks[b]), pre - b * bt if b == pre // bt else 0
            for t in (self.k, self.v):
                t[i, :, max(lo, 0):] = bad
            if b > pre // bt or pre % bt == 0:
                self.ks[i] = self.vs[i] = math.nan

    def objects(self):
        starts = [0]
        for n in self.news:
            starts.append(starts[-1] + n)
        even = len(set(self.news)) == 1
        cache = serve.Kv8Cache.from_buffers(self.k, self.v, self.ks, self.vs, self.fmt)
        batch = serve.Kv8Batch(self.table, self.lengths, starts[-1],
                               row_start=None if even else torch.tensor(starts, dtype=torch.int32, device=DEV), max_new=max(self.news))
        return cache, batch, serve.Kv8Prefix(self.blocks, self.length), starts

    def run(self, **kw):
        cache, batch, prefix, _ = self.objects()
        return cache.prefix_attention(batch, prefix, self.q, token_mask=self.mask, **kw)

    def read(self, ids, count):
        t = torch.arange(count, device=DEV)
        ids = ids.long()[t // self.bt]
        key = values(self.k[ids, :, t % self.bt], self.fmt) * self.ks[ids].double()[..., None]
        val = values(self.v[ids, :, t % self.bt], self.fmt) * self.vs[ids].double()[..., None]
        return key.transpose(0, 1), val.transpose(0, 1), self.vs[ids].double().t()   # [nkv, T, ...]

    def check(self, o, lse, pre=None, gone=()):
        pre = self.pre if pre is None else pre
        pk, pv, ps = self.read(self.blocks, pre)
        keep = torch.tensor([t // self.bt not in gone for t in range(pre)], dtype=torch.bool, device=DEV)
        pk, pv, ps = pk[:, keep], pv[:, keep], ps[:, keep]
        at = 0
        for b, (past, new) in enumerate(zip(self.own, self.news)):
            ok_, ov_, os_ = self.read(self.table[b], past + new)
            for i in range(new):
                see = torch.arange(past + new, device=DEV) <= past + i
                if self.mask is not None:
                    see &= self.mask[b, :past + new] != 0
                key, val, s = (torch.cat((x, y[:, see]), 1) for x, y in ((pk, ok_), (pv, ov_), (ps, os_)))
                got_o, got_l = o[at + i].double().view(self.nkv, self.group, self.hd), lse[at + i].double().view(self.nkv, self.group)
                if key.shape[1] == 0:
                    assert (got_o == 0).all() and (got_l == -math.inf).all()
                    continue
                q = self.q[at + i].double().view(self.nkv, self.group, self.hd)
                z = torch.einsum("hgd,htd->hgt", q, key) * self.scale
                want_l = torch.logsumexp(z, -1)
                p = torch.exp(z - want_l[..., None])
                want_o = torch.einsum("hgt,htd->hgd", p, val)
                mags = torch.einsum("hgd,htd->hgt", q.abs(), key.abs()).amax(-1) * self.scale
                ds = mags * (self.hd + 8) * 2.0 ** -23 + (mags * 1.45 + 150) * 2.0 ** -23
                spread = torch.einsum("hgt,htd->hgd", p, val.abs())
                flush = (p * s[:, None]).amax(-1) * key.shape[1] * 512 * 2.0 ** -35
                gone_v = torch.einsum("hgt,htd->hgd", p * (s < 2.0 ** -90)[:, None], val.abs())
                tol = 2 * (2.0 ** -11 + 2 * ds)[..., None] * spread + flush[..., None] + gone_v
                tol = tol + torch.finfo(torch.bfloat16).eps / 2 * (want_o.abs() + tol) + 1e-30
                assert ((got_o - want_o).abs() <= tol).all(), (b, i, ((got_o - want_o).abs() - tol).max().item())
                tol_l = ds + (8 + key.shape[1] / 32) * 2.0 ** -23 + 2.0 ** -22 * want_l.abs()
                assert ((got_l - want_l).abs() <= tol_l).all(), (b, i, ((got_l - want_l).abs() - tol_l).max().item())
            at += new


SHAPES = [  # fmt, bt, nkv, group, hd, prefix, own, news
    ("int8", 16, 2, 7, 64, 777, [100, 0, 3], [1, 1, 1]),
    ("e4m3", 16, 1, 1, 128, 1, [0], [1]),
    ("int8", 32, 1, 3, 64, 0, [5, 17], [1, 1]),
    ("e4m3", 32, 2, 4, 128, 63, [0, 40], [2, 2]),
    ("int8", 64, 2, 4, 128, 64, [9], [1]),
    ("e4m3", 64, 1, 8, 64, 65, [0, 1, 2, 3], [1, 1, 1, 1]),
    ("int8", 128, 3, 2, 128, 128, [130, 7], [1, 1]),
    ("e4m3", 128, 1, 5, 128, 1000, [77], [3]),
    ("int8", 16, 8, 1, 64, 129, [30] * 3, [1] * 3),
    ("int8", 64, 2, 4, 128, 3001, [60, 5, 0, 31], [1, 9, 0, 40]),            # 100 to 200 rows a KV head, one sequence without any
    ("e4m3", 32, 1, 8, 128, 515, [9, 4], [37, 21]),                         # four tiles of rows
    ("int8", 16, 1, 6, 64, 97, [3] * 65, [1] * 65),                          # 390 rows
    ("e4m3", 16, 64, 1, 64, 200, [2, 2], [70, 70]),                          # more units than CTAs
    ("int8", 128, 40, 4, 64, 60, [2] * 3, [12] * 3),                         # units of one step
    ("int8", 64, 1, 4, 128, 20011, [33] * 2, [1] * 2),                       # many parts of a row
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_matches_the_formula(shape):
    c = Case(*shape, seed=len(str(shape)), room=1)
    c.check(*c.run())
    assert take_error() == 0


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("rows", [3, 50])
def test_values_of_very_different_scales(fmt, rows):
    """Blocks of V whose scales span 2^+-30, some of them 0: the weights of small ones still count in the sum of weights."""
    c = Case(fmt, 16, 2, 4, 64, 900, [20] * rows, [1] * rows, seed=3, spread=15.0)
    c.vs[c.blocks.long()[::5]] = 0.0
    c.check(*c.run())
    c.vs[c.blocks.long()] = 0.0
    c.check(*c.run())


@pytest.mark.parametrize("rows", [3, 50])
@pytest.mark.parametrize("power", [-119, -111, -91, -89, -60, 100])
def test_weights_count_whatever_the_values_scales(rows, power):
    """Weights over scales of V that are tiny or huge stay within 32 bits: lse does not depend on V."""
    c = Case("int8", 32, 2, 4, 64, 700, [40] * rows, [1] * rows, seed=17)
    _, lse = c.run()
    c.vs.fill_(2.0 ** power)
    o, got = c.run()
    c.check(o, got)
    assert ((got - lse).abs() <= 2.0 ** -15 * (1 + lse.abs())).all()


@pytest.mark.parametrize("q_amp", [0.0, 1e-3, 30.0, 1e4])
def test_scores_of_any_size(q_amp):
    """References that have to move, rows that see one token alone, and rows that weigh all alike."""
    c = Case("int8", 32, 2, 4, 128, 1500, [10] * 40, [1] * 40, seed=5, q_amp=q_amp)
    c.ks[c.blocks.long()] *= torch.linspace(0.01, 3.0, c.blocks.numel(), device=DEV)[:, None]   # ever larger scores
    if q_amp < 1e3:   # beyond, 32-bit scores differ by more than a weight
        c.check(*c.run())
    else:
        o, lse = c.run()
        assert torch.isfinite(o).all() and torch.isfinite(lse).all()


def test_queries_out_of_f16s_range():
    c = Case("int8", 64, 1, 4, 64, 300, [8] * 2, [1] * 2, seed=6)
    c.q = (c.q.float() * torch.tensor([1e-30, 1e30, 1.0, 1e-39], device=DEV)[None, :, None]).to(torch.bfloat16)
    c.scale = 1e-30
    o, lse = c.run(scale=1e-30)
    q = c.q.clone()
    c.check(o, lse)
    c.q = q
    c.q[0, 0, 5] = math.nan
    o, lse = c.run(scale=1e-30)
    assert torch.isnan(o[0, 0]).all() and torch.isfinite(o[0, 1:]).all() and torch.isfinite(o[1]).all()


def test_own_tokens_that_are_masked():
    c = Case("e4m3", 16, 2, 3, 64, 70, [40, 12, 0], [2, 2, 2], seed=7)
    c.mask = torch.ones(3, c.table.shape[1] * 16, device=DEV, dtype=torch.uint8)
    c.mask[0, ::3] = 0
    c.mask[1] = 0
    c.check(*c.run())
    c.length.zero_()   # nothing at all is left for sequence 1
    c.check(*c.run(), pre=0)


def test_a_visible_nan_code_is_seen():
    c = Case("e4m3", 32, 1, 2, 64, 200, [5] * 2, [1] * 2, seed=8)
    c.v[c.blocks[3].item(), 0, 7, 9] = 0x7F
    o, _ = c.run()
    assert torch.isnan(o[:, :, 9]).all() and torch.isfinite(o[:, :, :9]).all() and torch.isfinite(o[:, :, 10:]).all()


@pytest.mark.parametrize("rows", [2, 60])
def test_bad_blocks_and_lengths(rows):
    """Block ids outside the pool are skipped, lengths that the blocks do not hold count as none; both are reported."""
    c = Case("int8", 16, 2, 4, 64, 333, [20] * rows, [1] * rows, seed=9)
    take_error()
    good = c.blocks.clone()
    for bad in (-1, -2, c.k.shape[0], 2 ** 31 - 1, -2 ** 31):
        c.blocks[4], c.blocks[20] = bad, bad
        o, lse = c.run()
        c.blocks.copy_(good)
        assert take_error() == 2
        c.check(o, lse, gone=(4, 20))
    for length in (-1, c.blocks.numel() * 16 + 1, -2 ** 31):
        c.length.fill_(length)
        o, lse = c.run()
        assert take_error() == 2
        c.check(o, lse, pre=0)
    c.length.fill_(333)
    c.check(*c.run())
    assert take_error() == 0


def test_sequences_that_do_not_fit_and_rows_behind_the_last():
    """What belongs to no sequence, or to one that its table cannot hold, is left as it was."""
    c = Case("int8", 32, 1, 4, 64, 150, [10, 11, 12], [1, 3, 2], seed=10)
    cache, _, prefix, starts = c.objects()
    take_error()
    rows = starts[-1] + 4
    q = torch.cat((c.q, torch.full((4, *c.q.shape[1:]), math.nan, device=DEV, dtype=torch.bfloat16)))
    lengths = torch.tensor([10, 1 << 20, 12], dtype=torch.int32, device=DEV)
    batch = serve.Kv8Batch(c.table, lengths, rows, row_start=torch.tensor(starts, dtype=torch.int32, device=DEV), max_new=3)
    out = torch.full(q.shape, 7.0, device=DEV, dtype=torch.bfloat16)
    o, lse = cache.prefix_attention(batch, prefix, q, out=out)
    assert o is out and take_error() == 2
    assert (out[1:4] == 7).all() and (out[6:] == 7).all()
    want, want_l = c.run()
    assert torch.equal(out[[0, 4, 5]], want[[0, 4, 5]]) and torch.equal(lse[[0, 4, 5]], want_l[[0, 4, 5]])


def test_is_attention_over_the_whole():
    """The prefix as every sequence's own first blocks, through the plain call."""
    c = Case("int8", 64, 2, 4, 128, 640, [70, 1, 128], [1] * 3, seed=11)
    o, lse = c.run()
    whole = torch.cat((c.blocks.expand(3, -1), c.table), 1).contiguous()
    cache, *_ = c.objects()
    o2, lse2 = cache.attention(serve.Kv8Batch(whole, c.lengths + 640, 3), c.q)
    assert (o.float() - o2.float()).abs().max() <= 2 ** -7 * o2.float().abs().max()
    assert (lse - lse2).abs().max() <= 2 ** -19 * lse2.abs().max()


def test_no_rows():
    c = Case("int8", 16, 1, 1, 64, 20, [3, 3], [1, 1], seed=12)
    cache, _, prefix, _ = c.objects()
    batch = serve.Kv8Batch(c.table, c.lengths, 0, max_new=0)
    o, lse = cache.prefix_attention(batch, prefix, c.q[:0])
    assert o.shape == (0, 1, 64) and lse.shape == (0, 1)
    c.run()
    assert take_error() == 0


def test_graphs_follow_the_lengths_and_do_not_share():
    """Two captured calls replay side by side while their prefixes and sequences grow."""
    cases = [Case("int8", 32, 2, 4, 128, 900, [200] * 3, [1] * 3, seed=13), Case("e4m3", 64, 1, 8, 64, 2000, [90] * 20, [2] * 20, seed=14)]
    side, graphs, outs, kept = [torch.cuda.Stream() for _ in cases], [], [], []
    for c, st in zip(cases, side):
        c.run()
        kept.append(c.objects())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            cache, batch, prefix, _ = kept[-1]
            outs.append(cache.prefix_attention(batch, prefix, c.q))
        graphs.append(g)
    for turn in range(6):
        want = []
        for c in cases:
            c.length.fill_(c.pre - 150 * turn if turn < 5 else 0)
            c.lengths.fill_(c.own[0] - 13 * turn)
            want.append(c.run())
        torch.cuda.synchronize()
        for g, st in zip(graphs, side):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
    assert take_error() == 0


def test_a_prefix_without_blocks_waits_for_what_ran_before():
    """Nothing of the call may start before the kernel that writes its queries has ended."""
    c = Case("int8", 32, 2, 4, 64, 0, [300] * 64, [1] * 64, seed=16)
    cache, batch, prefix, _ = c.objects()
    assert prefix.blocks.numel() == 0
    want = c.run()
    c.check(*want)
    big = torch.zeros(1 << 26, device=DEV, dtype=torch.bfloat16)
    q = c.q.contiguous()
    n = q.numel()
    for _ in range(20):
        big.zero_()
        big[-n:].copy_(q.flatten())
        got = cache.prefix_attention(batch, prefix, big[-n:].view(q.shape))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert take_error() == 0


def test_another_stream():
    c = Case("int8", 16, 2, 7, 64, 500, [33] * 4, [1] * 4, seed=15)
    want = c.run()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = [c.run() for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[0]) and torch.equal(l, want[1]) for o, l in got)
