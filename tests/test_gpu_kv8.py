"""The 8-bit key/value cache (glt_kv8_append, glt_kv8_attention, glt_kv8_read)
against plain 64-bit forms.

Append and read are held to equality: the rule of the format fixes every bit
(a scale is the 32-bit quotient of a maximum, a code the nearest to a 32-bit
quotient).  Attention's tolerance is derived in `attention_ref`."""
import math

import pytest
import torch

from glt_b200 import _lib, serve

pytestmark = pytest.mark.gpu
TOP = {"int8": 127.0, "e4m3": 448.0}
DEV = "cuda"


def encode(y32, fmt):
    """Nearest code's value of a 32-bit quotient."""
    if fmt == "int8":
        return y32.round().clamp(-127, 127).double()
    return y32.clamp(-448, 448).to(torch.float8_e4m3fn).double()


class RefCache:
    """Per (sequence, block, head): code values and the scale, grown token block by token block."""

    def __init__(self, fmt, bt, nkv, hd):
        self.fmt, self.bt, self.nkv, self.hd = fmt, bt, nkv, hd
        self.codes, self.scale, self.held = {}, {}, {}

    def append(self, b, rows):
        """rows: [n, nkv, hd] bf16 on the CPU."""
        past = self.held.get(b, 0)
        at = 0
        while at < rows.shape[0]:
            blk, lo = (past + at) // self.bt, (past + at) % self.bt
            n = min(self.bt - lo, rows.shape[0] - at)
            x = rows[at:at + n].float()
            fin = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
            s1 = (fin.amax((0, 2)).double() / TOP[self.fmt]).float()
            if lo:
                s0, old = self.scale[b, blk], self.codes[b, blk]
                s1 = torch.maximum(s0, s1)
                val = (old * s0.double()[None, :, None]).float()
                grew = (s1 > s0)[None, :, None]
                old = torch.where(grew, encode(quot(val, s1), self.fmt), old)
            else:
                old = torch.zeros(0, self.nkv, self.hd, dtype=torch.float64)
            y = quot(torch.nan_to_num(x, nan=0.0, posinf=math.inf, neginf=-math.inf), s1)
            self.codes[b, blk] = torch.cat((old, encode(y, self.fmt)))
            self.scale[b, blk] = s1
            at += n
        self.held[b] = past + rows.shape[0]

    def values(self, b):
        out = [self.codes[b, k] * self.scale[b, k].double()[None, :, None]
               for k in range(-(-self.held.get(b, 0) // self.bt))]
        return torch.cat(out) if out else torch.zeros(0, self.nkv, self.hd, dtype=torch.float64)


def quot(x, s):
    y = (x.double() / s.double()[None, :, None]).float()
    return torch.where(s[None, :, None] > 0, y, torch.zeros_like(y))


def garbage_cache(num_blocks, bt, nkv, hd, fmt):
    """A cache whose unwritten codes and scales are NaN patterns."""
    c = serve.Kv8Cache(num_blocks, bt, nkv, hd, fmt)
    for t in (c.k, c.v):
        t.fill_(0xFF)
    for t in (c.k_scale, c.v_scale):
        t.fill_(math.nan)
    return c


def tables(seqs, maxb, num_blocks, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(num_blocks, generator=g)[:seqs * maxb].view(seqs, maxb).to(torch.int32).to(DEV)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def rows_of(g, n, nkv, hd, amp=1.0):
    return (torch.randn(n, nkv, hd, generator=g) * amp).to(torch.bfloat16)


def attention_ref(q, k, v, past, scale, window=0, mask=None):
    """q [n, nh, hd], k/v [T, nkv, hd] (fp64) -> o, lse, tolerance of o, tolerance of lse.

    The kernel may round a probability to f16 (relative 2^-11) and its scores carry the error of
    hd products and a scale in 32 bits: |ds| <= (hd + 8) 2^-24 sum|q||k| scale (and twice that
    where the tensor core truncates), which scales a probability by exp(ds).  So
    |do| <= (2^-11 + 2 ds) sum p|v| (1 + small), doubled for the normalisation, plus bf16's 2^-9 |o|."""
    n, nh, hd = q.shape
    T, nkv, _ = k.shape
    group = nh // nkv
    o = torch.zeros(n, nh, hd, dtype=torch.float64)
    lse = torch.full((n, nh), -math.inf, dtype=torch.float64)
    otol = torch.zeros(n, nh, hd, dtype=torch.float64)
    ltol = torch.zeros(n, nh, dtype=torch.float64)
    t = torch.arange(T)
    for i in range(n):
        see = t <= past + i
        if window:
            see &= t > past + i - window
        if mask is not None:
            see &= mask[:T].bool()
        idx = see.nonzero()[:, 0]
        if not idx.numel():
            continue
        for h in range(nh):
            kk, vv, qq = k[idx, h // group], v[idx, h // group], q[i, h].double()
            z = kk @ qq * scale
            lse[i, h] = torch.logsumexp(z, 0)
            p = torch.exp(z - lse[i, h])
            o[i, h] = p @ vv
            ds = (kk.abs() @ qq.abs()).max() * scale * (hd + 8) * 2.0 ** -23
            otol[i, h] = 2 * (2.0 ** -11 + 2 * ds) * (p @ vv.abs()) + 2.0 ** -8 * o[i, h].abs() + 1e-30
            ltol[i, h] = ds + (4 + idx.numel() / 32) * 2.0 ** -23 + 2.0 ** -22 * lse[i, h].abs()
    return o, lse, otol, ltol


def check(o, lse, ref, what):
    o_ref, lse_ref, otol, ltol = ref
    bad = (o.double().cpu() - o_ref).abs() > otol
    assert not bad.any(), f"{what}: o off by {((o.double().cpu() - o_ref).abs() - otol).max():.3e} past its tolerance"
    lse = lse.double().cpu()
    empty = lse_ref == -math.inf
    assert torch.equal(lse == -math.inf, empty), f"{what}: empty rows"
    assert (o.double().cpu()[empty] == 0).all(), f"{what}: empty rows must be 0"
    assert ((lse - lse_ref).abs()[~empty] <= ltol[~empty]).all(), f"{what}: lse"


class Session:
    """Drives a cache and its reference through steps of packed qkv rows."""

    def __init__(self, fmt, bt, nkv, group, hd, seqs, room, seed=0):
        self.fmt, self.bt, self.nkv, self.nh, self.hd, self.seqs = fmt, bt, nkv, nkv * group, hd, seqs
        self.maxb = -(-room // bt)
        self.cache = garbage_cache(seqs * self.maxb + 5, bt, nkv, hd, fmt)
        self.table = tables(seqs, self.maxb, self.cache.num_blocks, seed)
        self.g = torch.Generator().manual_seed(seed + 1)
        self.ref = {s: RefCache(fmt, bt, nkv, hd) for s in "kv"}
        self.lens = [0] * seqs

    def step(self, news, amp=1.0, **kw):
        rows = sum(news)
        # [q | k | v] rows with 8 columns to spare, as a projection would leave them
        W = (self.nh + 2 * self.nkv) * self.hd
        qkv = torch.zeros(rows, W + 8, dtype=torch.bfloat16)
        qkv[:, :W] = (torch.randn(rows, W, generator=self.g) * amp).to(torch.bfloat16)
        dev = qkv.to(DEV)
        a, b = self.nh * self.hd, (self.nh + self.nkv) * self.hd
        q, k, v = dev[:, :a], dev[:, a:b], dev[:, b:W]
        starts = [0]
        for n in news:
            starts.append(starts[-1] + n)
        even = len(set(news)) == 1
        batch = serve.Kv8Batch(self.table, i32(self.lens), rows, row_start=None if even else i32(starts),
                               max_new=max(news))
        self.cache.append(batch, k.unflatten(1, (self.nkv, self.hd)), v.unflatten(1, (self.nkv, self.hd)))
        for s in range(self.seqs):
            sl = slice(starts[s], starts[s + 1])
            self.ref["k"].append(s, qkv[sl, a:b].reshape(-1, self.nkv, self.hd))
            self.ref["v"].append(s, qkv[sl, b:W].reshape(-1, self.nkv, self.hd))
        mask = kw.pop("mask", None)
        o, lse = self.cache.attention(batch, q.unflatten(1, (self.nh, self.hd)),
                                      token_mask=None if mask is None else mask.to(DEV), **kw)
        scale = kw.get("scale") or 1 / math.sqrt(self.hd)
        for s in range(self.seqs):
            sl = slice(starts[s], starts[s + 1])
            ref = attention_ref(qkv[sl, :a].reshape(-1, self.nh, self.hd), self.ref["k"].values(s),
                                self.ref["v"].values(s), self.lens[s], scale, kw.get("window", 0),
                                None if mask is None else mask[s])
            check(o[sl], lse[sl], ref, f"sequence {s}")
        self.batch = batch
        self.lens = [x + n for x, n in zip(self.lens, news)]
        code = _lib.C.c_uint()
        assert _lib.lib.glt_device_error(_lib.C.byref(code)) == 0 and code.value == 0

    def check_values(self):
        top = max(self.lens)
        k, v = self.cache.read(self.batch, None, top + 3)
        for s in range(self.seqs):
            for got, want in ((k, self.ref["k"]), (v, self.ref["v"])):
                assert torch.equal(got[s, :self.lens[s]].cpu(), want.values(s).float())
                assert (got[s, self.lens[s]:] == 0).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bt,nkv,group,hd", [(16, 2, 7, 64), (32, 1, 1, 128), (64, 2, 4, 128), (128, 3, 2, 64),
                                             (16, 1, 8, 128), (128, 1, 5, 128)])
def test_prompt_then_single_tokens(fmt, bt, nkv, group, hd):
    """A prompt of uneven lengths (one of them empty), then single tokens across block edges."""
    s = Session(fmt, bt, nkv, group, hd, seqs=4, room=200, seed=bt + hd)
    s.step([37, 1, 0, 130])
    s.check_values()
    for i in range(4):
        s.step([1, 1, 1, 1], amp=1.0 + i)   # growing values: the scales of part-filled blocks rise
        s.check_values()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("news", [[3, 3], [1, 9], [2, 0], [17, 40]])
def test_several_new_tokens_with_window_and_scale(fmt, news):
    s = Session(fmt, 32, 2, 3, 64, seqs=2, room=400, seed=5)
    s.step([150, 61])
    s.step(news, window=33, scale=0.37)
    s.step(news, window=1)
    s.check_values()


@pytest.mark.parametrize("length", [0, 1, 15, 16, 31, 32, 33, 63, 64, 127, 128, 129, 511, 1000])
def test_lengths_around_tile_edges(length):
    s = Session("int8", 16, 1, 4, 128, seqs=1, room=1010, seed=length)
    if length:
        s.step([length], window=7)
    s.step([1])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_masks_that_leave_rows_empty(fmt):
    s = Session(fmt, 16, 2, 2, 64, seqs=3, room=160, seed=9)
    width = s.maxb * 16
    g = torch.Generator().manual_seed(3)
    mask = (torch.rand(3, width + 5, generator=g) > 0.4).to(torch.uint8) * 255
    mask[1] = 0                      # nothing to see at all
    mask[2, :140] = 0                # a window that holds nothing
    s.step([140, 20, 140], mask=mask[:, :width])
    s.step([2, 2, 2], mask=mask, window=2)
    s.step([1, 1, 1], mask=mask[:, :width].bool())


def test_large_and_small_magnitudes():
    """Blocks whose scales differ by forty orders of magnitude, zero blocks, queries of any size."""
    for amp in (1e-30, 1e18):
        s = Session("int8", 16, 1, 4, 64, seqs=1, room=200, seed=int(math.log10(amp)) + 50)
        for a in (1.0, amp, 0.0, 1.0):
            s.step([16], amp=a, scale=1e-3 if amp < 1 else 1e-36)
        s.check_values()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("power", [0, 100, -50, -55, -62, -110])
def test_codes_are_those_of_a_division(fmt, power):
    """Every bf16 mantissa under a maximum of every mantissa (a head each), quotients that meet the codes' boundaries
    among them, and the codes of a block whose scale rises: equal to rounding the 32-bit quotient."""
    nkv, hd = 128, 64
    cache = garbage_cache(3, 128, nkv, hd, fmt)
    table = torch.tensor([[2]], dtype=torch.int32, device=DEV)
    ref = {s: RefCache(fmt, 128, nkv, hd) for s in "kv"}
    g = torch.Generator().manual_seed(power + 200)
    past = 0
    for n, rise in ((100, 1.0), (28, 1.37)):
        i = torch.arange(n * hd)
        x = (1 + (i % 128) / 128) * torch.exp2(-((i // 128) % 14).float() - 1)
        x = x[torch.randperm(n * hd, generator=g)].view(n, 1, hd) * torch.randint(0, 2, (n, 1, hd), generator=g).mul(2).sub(1)
        x = x.repeat(1, nkv, 1)
        x[n // 2, :, 5] = 1 + torch.arange(nkv) / nkv   # the largest magnitude
        x = (x * rise * 2.0 ** power).to(torch.bfloat16)
        batch = serve.Kv8Batch(table, i32([past]), n, max_new=n)
        cache.append(batch, x.to(DEV), -x.to(DEV))
        ref["k"].append(0, x)
        ref["v"].append(0, -x)
        past += n
        k, v = cache.read(batch, None, past)
        assert torch.equal(k[0].cpu(), ref["k"].values(0).float())
        assert torch.equal(v[0].cpu(), ref["v"].values(0).float())


def test_non_finite_keys_saturate_and_nan_is_zero():
    for fmt in ("int8", "e4m3"):
        c = garbage_cache(3, 16, 1, 64, fmt)
        table, rows = i32([[2]]), torch.randn(3, 1, 64).to(torch.bfloat16)
        rows[0, 0, 0], rows[1, 0, 1], rows[2, 0, 2] = math.inf, -math.inf, math.nan
        batch = serve.Kv8Batch(table, i32([0]), 3)
        c.append(batch, rows.to(DEV), rows.to(DEV))
        k, v = c.read(batch, None, 3)
        ref = RefCache(fmt, 16, 1, 64)
        ref.append(0, rows)
        assert torch.equal(k[0].cpu(), ref.values(0).float()) and torch.equal(v, k)
        assert k[0, 2, 0, 2] == 0 and k[0, 0, 0, 0] == rows[torch.isfinite(rows)].abs().max().float()


def test_offsets_past_32_bits():
    """Blocks that start beyond 2^32 bytes into the pool."""
    n = (1 << 32) // (128 * 128) + 40
    c = serve.Kv8Cache(n, 128, 1, 128, "int8")
    s = Session("int8", 128, 1, 4, 128, seqs=2, room=300, seed=2)
    s.cache, s.table = c, i32([[n - 1, n - 7, n - 3], [n - 2, 5, n - 9]])
    s.step([290, 200])
    s.step([1, 1])
    s.check_values()
    del s, c
    torch.cuda.empty_cache()


def test_long_cache_of_one_sequence():
    """More tokens than any one CTA takes: the partial results are joined."""
    hd, nkv, group, T = 64, 2, 7, 9001
    s = Session("e4m3", 64, nkv, group, hd, seqs=1, room=T + 64, seed=4)
    s.step([T], window=1)
    s.step([1])
    s.step([3], window=5000)


def test_side_stream_and_repeated_calls_agree():
    s = Session("int8", 32, 2, 4, 128, seqs=5, room=3000, seed=6)
    s.step([2900, 1, 700, 33, 64], window=1)
    q = torch.randn(5, 8, 128, device=DEV).to(torch.bfloat16)
    batch = serve.Kv8Batch(s.table, i32([x - 1 for x in s.lens]), 5)
    a = s.cache.attention(batch, q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b = s.cache.attention(batch, q)
    side.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_cuda_graph_replay_follows_lengths():
    """The lengths are read on the device: one captured step serves every position."""
    s = Session("int8", 16, 1, 4, 64, seqs=2, room=100, seed=8)
    s.step([40, 7])
    lens, q = i32(s.lens), torch.randn(2, 4, 64, device=DEV).to(torch.bfloat16)
    kv = torch.randn(2, 2, 1, 64, device=DEV).to(torch.bfloat16)
    batch = serve.Kv8Batch(s.table, lens, 2)
    s.cache.append(batch, kv[0], kv[1])
    s.cache.attention(batch, q)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.cache.append(batch, kv[0], kv[1])
        o, lse = s.cache.attention(batch, q)
    for _ in range(3):
        g.replay()
        want = s.cache.attention(batch, q)
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
        lens += 1


def device_error():
    code = _lib.C.c_uint()
    _lib.lib.glt_device_error(_lib.C.byref(code))
    return code.value


def test_bad_device_values_set_the_error_word():
    """Out-of-range lengths, rows and block ids: nothing is read or written there."""
    c = garbage_cache(4, 16, 1, 64, "int8")
    x = torch.randn(2, 1, 64, device=DEV).to(torch.bfloat16)
    q = torch.randn(2, 2, 64, device=DEV).to(torch.bfloat16)
    device_error()
    for table, lens, starts in (([[0, 1], [2, 3]], [-1, 0], None), ([[0, 1], [2, 3]], [32, 0], None),
                                ([[4, 1], [2, 3]], [0, 0], None), ([[-1, 1], [2, 3]], [0, 0], None),
                                ([[0, 1], [2, 3]], [0, 0], [0, 3, 2]), ([[0, 1], [2, 3]], [0, 0], [-1, 1, 2])):
        before = [t.clone() for t in (c.k, c.v)]
        batch = serve.Kv8Batch(i32(table), i32(lens), 2, row_start=None if starts is None else i32(starts), max_new=1)
        c.append(batch, x, x)
        assert device_error() == 2
        for t, old in zip((c.k, c.v), before):
            assert torch.equal(t[:2], old[:2])      # sequence 0 is the faulty one
        out = torch.full((2, 2, 64), 7.0, device=DEV, dtype=torch.bfloat16)
        c.attention(batch, q, out=out)
        assert device_error() == 2
        if starts is None:
            assert torch.isfinite(out[1].float()).all() and (out[1] != 7).any()
    c.read(serve.Kv8Batch(i32([[9, 1]]), i32([3]), 0, max_new=0), None, 3)
    assert device_error() == 2


def test_nan_queries_give_nan_in_their_rows_only():
    s = Session("int8", 32, 1, 2, 64, seqs=2, room=400, seed=11)
    s.step([300, 300], window=1)
    q = torch.randn(2, 2, 64, device=DEV).to(torch.bfloat16)
    batch = serve.Kv8Batch(s.table, i32([x - 1 for x in s.lens]), 2)
    want = s.cache.attention(batch, q)
    bad = q.clone()
    bad[0, 1, 3] = math.nan
    o, lse = s.cache.attention(batch, bad)
    assert torch.isnan(o[0, 1]).all() and torch.isnan(lse[0, 1])
    for r, h in ((0, 0), (1, 0), (1, 1)):
        assert torch.equal(o[r, h], want[0][r, h]) and lse[r, h] == want[1][r, h]
