"""Cases that measure the operators for serving many users with one baked model, with their plain forms.

Three operators: products in 8-bit integers with a scale for each token and each channel (the
tokens are quantised in the call, after their RMSNorm where a case has one), attention of a batch
of sequences that share a long prefix over the 8-bit cache, and attention over that cache with a
sliding window and a few first tokens that stay visible.  ``own`` selects what ``run`` computes
with: elementary torch operations in 32 bits, or the library's entry points in ``glt_b200.serve``.
"""
import math
import random

import torch

own = False

DEV = "cuda"
INT8_MAX, E4M3_MAX = 127.0, 448.0
EPS = 1e-6


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # single token through the Qwen2.5-0.5B down projection: launch latency counts
        w8("w8_small", m=1, n=896, k=4864, resid=True),
        # one token of eight users through the Llama-3-8B norm, gate and up projections
        w8("w8_gate_up", m=8, n=28672, k=4096, norm=True),
        # draft tokens of a batch through a width that fits no tile, logits kept in 32 bits
        w8("w8_drafts", m=60, n=32001, k=4097, out="fp32"),
        # a prompt through the Llama-3-8B down projection, with the residual
        w8("w8_prompt_down", m=2047, n=4096, k=14336, resid=True),
        # a batch of prompts through the Llama-3-8B norm, gate and up projections
        w8("w8_prompts_gate_up", m=8192, n=28672, k=4096, norm=True),
        # a few users of the Qwen2.5-0.5B head layout behind a short common instruction
        prefix("prefix_few", fmt="int8", bt=16, seqs=3, pre=777, ctx=100, nkv=2, group=7, hd=64),
        # a serving batch behind one system prompt on the Llama-3-8B head layout, users at different positions
        prefix("prefix_batch", fmt="int8", bt=64, seqs=64, pre=8193, ctx=1023, ragged=True, nkv=8, group=4, hd=128),
        # many questions about one long document
        prefix("prefix_document", fmt="e4m3", bt=128, seqs=128, pre=65537, ctx=301, ragged=True, nkv=8, group=4, hd=128),
        # every user's question enters at once behind the prompt
        prefix("prefix_questions", fmt="e4m3", bt=32, seqs=16, pre=4099, ctx=9, ragged=True, new=37, nkv=4, group=8,
               hd=128, masked=True),
        # one user's endless stream on the Qwen2.5-0.5B head layout
        sinks("sinks_one_user", fmt="int8", bt=16, seqs=1, ctx=20011, nkv=2, group=7, hd=64, window=1023, first=4),
        # a batch of streams of very different ages on the Llama-3-8B head layout
        sinks("sinks_batch", fmt="int8", bt=64, seqs=48, ctx=60001, ragged=True, nkv=8, group=4, hd=128, window=4096,
              first=5),
        # five draft tokens a stream, checked at once, dropped tokens among them
        sinks("sinks_drafts", fmt="e4m3", bt=32, seqs=12, ctx=9001, ragged=True, new=5, nkv=4, group=8, hd=128,
              window=2047, first=67, masked=True),
    ]


def w8(name, **kw):
    return dict(dict(name=name, op="w8", norm=False, resid=False, out="bf16"), **kw)


def prefix(name, **kw):
    return dict(dict(name=name, op="prefix", ragged=False, new=1, masked=False), **kw)


def sinks(name, **kw):
    return dict(dict(name=name, op="sinks", ragged=False, new=1, masked=False), **kw)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _odd(rng, lo, hi):
    return 2 * (_log(rng, lo, hi) // 2) + 1


def draw(rng):
    op = rng.choice(["w8", "prefix", "sinks"])
    if op == "w8":
        c = w8("", m=_log(rng, 1, 8192), n=_odd(rng, 64, 32001), k=_log(rng, 64, 14336), norm=rng.random() < 0.5,
               resid=rng.random() < 0.5, out=rng.choice(["bf16", "fp32"]))
        if rng.random() < 0.5:
            c["n"], c["k"] = max(64, c["n"] // 64 * 64), max(64, c["k"] // 64 * 64)
        while c["m"] * c["n"] * c["k"] > 8192 * 28672 * 4096:
            c["m"] = (c["m"] + 1) // 2
    else:
        hd, nkv, group = rng.choice([64, 128]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 6, 7, 8])
        fmt, bt = rng.choice(["int8", "e4m3"]), rng.choice([16, 32, 64, 128])
        common = dict(fmt=fmt, bt=bt, nkv=nkv, group=group, hd=hd, ragged=rng.random() < 0.6,
                      masked=rng.random() < 0.3)
        if op == "prefix":
            seqs, new = _log(rng, 1, 128), rng.choice([1, 1, 1, 2, 5, 37])
            while seqs * new > 600:
                seqs //= 2
            pre = _odd(rng, 15, min(65537, 128 * 65537 * 32 * 128 // (seqs * new * nkv * group * hd)))
            c = prefix("", seqs=seqs, new=new, pre=pre, ctx=_odd(rng, 1, min(2047, 65537 // seqs)), **common)
        else:
            seqs, new = _log(rng, 1, 48), rng.choice([1, 1, 1, 2, 3, 5, 7])
            window = _odd(rng, 1, min(8191, 48 * 4096 // (seqs * new)))
            c = sinks("", seqs=seqs, new=new, window=window, first=_log(rng, 1, 128), ctx=_odd(rng, 1, 60001), **common)
    del c["name"]
    return c


# --------------------------------------------------------------------------- sizes
def lengths_of(c):
    """A sequence's own tokens in the cache before the call: ctx for all, or spread from none to ctx."""
    n = c["seqs"]
    if not c["ragged"]:
        return [c["ctx"]] * n
    r = random.Random(n * 1000003 + c["ctx"])
    return [c["ctx"] if i == 0 else int((c["ctx"] + 1) * r.random() ** 1.5) for i in range(n)]


def _seen(c):
    """(tokens that some query of the step sees, pairs of a query and a token it sees), summed over the sequences."""
    seen = pairs = 0
    for past in lengths_of(c):
        if c["op"] == "prefix":
            seen += past + c["new"]
            pairs += sum(c["pre"] + past + i + 1 for i in range(c["new"]))
            continue
        low = max(0, past - c["window"] + 1)
        seen += past + c["new"] - low + min(low, c["first"])
        for i in range(c["new"]):
            low = max(0, past + i - c["window"] + 1)
            pairs += past + i + 1 - low + min(low, c["first"])
    return seen + (c["pre"] if c["op"] == "prefix" else 0), pairs


def work(c):
    if c["op"] == "w8":
        m, n, k = c["m"], c["n"], c["k"]
        byt = 2 * m * k + n * k + 4 * n + m * n * (2 if c["out"] == "bf16" else 4)
        byt += (2 * m * n if c["resid"] else 0) + (2 * k if c["norm"] else 0)
        return {"bytes": byt, "flops": 2 * m * n * k}
    per, nh, hd = c["nkv"] * c["hd"], c["nkv"] * c["group"], c["hd"]
    seen, pairs = _seen(c)
    rows = c["seqs"] * c["new"]
    byt = 2 * seen * per + 8 * c["nkv"] * (seen // c["bt"] + c["seqs"]) + 4 * rows * nh * hd + 4 * rows * nh
    if c["masked"]:
        byt += seen - (c["pre"] if c["op"] == "prefix" else 0)
    return {"bytes": byt, "flops": 4 * pairs * nh * hd}


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _prepare_w8(c, seed):
    g = _gen(seed)
    m, n, k = c["m"], c["n"], c["k"]
    # activations have a few strong channels, and tokens differ in size
    x = torch.randn(m, k, device=DEV, generator=g) * torch.exp(torch.randn(m, 1, device=DEV, generator=g))
    x[:, :: max(1, k // 6)] *= 8.0
    codes = torch.empty(n, k, dtype=torch.int8, device=DEV)
    scales = torch.empty(n, device=DEV)
    for i in range(0, n, 4096):
        w = torch.randn(min(4096, n - i), k, device=DEV, generator=g) * 0.02
        scales[i:i + 4096] = w.abs().amax(1) / INT8_MAX
        codes[i:i + 4096] = (w / scales[i:i + 4096, None]).round().clamp(-127, 127).to(torch.int8)
    s = dict(case=c, x=x.to(torch.bfloat16), codes=codes, scales=scales, resid=None, norm=None)
    if c["resid"]:
        s["resid"] = torch.randn(m, n, device=DEV, generator=g).to(torch.bfloat16)
    if c["norm"]:
        s["norm"] = (1 + 0.2 * torch.randn(k, device=DEV, generator=g)).to(torch.bfloat16)
    if own:
        from glt_b200 import serve
        s["weight"] = serve.W8Weight.from_codes(codes, scales)
        del s["codes"], s["scales"]
    return s


def _values(codes, fmt):
    return codes.float() - 128.0 if fmt == "int8" else codes.view(torch.float8_e4m3fn).float()


def _fill(pool, scale, g, fmt, kind):
    """Random keys or values, quantised block by block: keys have a few strong channels."""
    nb, nkv, bt, hd = pool.shape
    top = INT8_MAX if fmt == "int8" else E4M3_MAX
    amp = torch.ones(nkv, 1, hd, device=DEV)
    if kind == "k":
        amp[:, :, :: hd // 4] = 4.0
    for i in range(0, nb, 1024):
        x = torch.randn(min(1024, nb - i), nkv, bt, hd, device=DEV, generator=g) * amp
        s = x.abs().amax((2, 3), keepdim=True) / top
        y = x / s
        if fmt == "int8":
            pool[i:i + 1024] = (y.round().clamp(-127, 127) + 128).to(torch.uint8)
        else:
            pool[i:i + 1024] = y.clamp(-top, top).to(torch.float8_e4m3fn).view(torch.uint8)
        scale[i:i + 1024] = s[:, :, 0, 0]


def _held(c):
    """The blocks that each sequence holds: all of its own, or those of its first tokens and its window."""
    bt, out = c["bt"], []
    for past in lengths_of(c):
        last = (past + c["new"] - 1) // bt
        if c["op"] == "prefix":
            out.append(list(range(last + 1)))
        else:
            low = max(0, past - c["window"] + 1) // bt
            early = range(min(low, (min(c["first"], past + c["new"]) - 1) // bt + 1))
            out.append(list(early) + list(range(low, last + 1)))
    return out


def _prepare_cache(c, seed):
    g = _gen(seed)
    held, pre_blocks = _held(c), -(-c.get("pre", 0) // c["bt"])
    nb, maxb = sum(len(h) for h in held) + pre_blocks + 3, max(h[-1] + 1 for h in held)
    perm = torch.randperm(nb, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((c["seqs"], maxb), -1, dtype=torch.int32)   # -1: a block that was given back
    at = pre_blocks
    for i, h in enumerate(held):
        table[i, h] = torch.tensor(perm[at:at + len(h)], dtype=torch.int32)
        at += len(h)
    shape = (nb, c["nkv"], c["bt"], c["hd"])
    k, v = (torch.empty(shape, dtype=torch.uint8, device=DEV) for _ in range(2))
    ks, vs = (torch.empty(nb, c["nkv"], device=DEV) for _ in range(2))
    _fill(k, ks, g, c["fmt"], "k")
    _fill(v, vs, g, c["fmt"], "v")
    rows, nh = c["seqs"] * c["new"], c["nkv"] * c["group"]
    # a packed row as the query/key/value projection leaves it: the queries are its first columns
    qkv = torch.randn(rows, (nh + 2 * c["nkv"]) * c["hd"], device=DEV, generator=g).to(torch.bfloat16)
    s = dict(case=c, k=k, v=v, ks=ks, vs=vs, table=table.to(DEV), rows=rows,
             lengths=torch.tensor(lengths_of(c), dtype=torch.int32, device=DEV),
             q=qkv[:, :nh * c["hd"]].view(rows, nh, c["hd"]), mask=None)
    if c["masked"]:
        s["mask"] = (torch.rand(c["seqs"], maxb * c["bt"], device=DEV, generator=g) > 0.25).to(torch.uint8)
    if c["op"] == "prefix":
        s["pre"] = torch.tensor(perm[:pre_blocks], dtype=torch.int32, device=DEV)
        s["pre_length"] = torch.tensor([c["pre"]], dtype=torch.int32, device=DEV)
    if own:
        from glt_b200 import serve
        s["cache"] = serve.Kv8Cache.from_buffers(k, v, ks, vs, c["fmt"])
        s["batch"] = serve.Kv8Batch(s["table"], s["lengths"], rows, max_new=c["new"])
        if c["op"] == "prefix":
            s["prefix"] = serve.Kv8Prefix(s["pre"], s["pre_length"])
    return s


def prepare(case, seed):
    return _prepare_w8(case, seed) if case["op"] == "w8" else _prepare_cache(case, seed)


# --------------------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return {"w8": _own_w8, "prefix": _own_prefix, "sinks": _own_sinks}[op](s)
    return _w8(s) if op == "w8" else _attention(s)


def _own_w8(s):
    return s["weight"].linear(s["x"], resid=s["resid"], norm=s["norm"], eps=EPS,
                              out_dtype=torch.bfloat16 if s["case"]["out"] == "bf16" else torch.float32)


def _own_prefix(s):
    return s["cache"].prefix_attention(s["batch"], s["prefix"], s["q"], token_mask=s["mask"])


def _own_sinks(s):
    c = s["case"]
    return s["cache"].attention(s["batch"], s["q"], window=c["window"], sinks=c["first"], token_mask=s["mask"])


def _w8(s):
    x = s["x"].float()
    if s["norm"] is not None:
        x = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * s["norm"].float()
    peak = x.abs().amax(1, keepdim=True)
    # a tensor divisor: a plain number would become a product with its rounded reciprocal
    scale = peak / torch.full_like(peak, INT8_MAX)
    codes = (x / torch.where(scale > 0, scale, torch.ones_like(scale))).round().clamp(-127, 127)
    y = torch.matmul(codes, s["codes"].float().t()) * s["scales"] * scale
    if s["resid"] is not None:
        y = y + s["resid"].float()
    return y.to(torch.bfloat16) if s["case"]["out"] == "bf16" else y


def _tokens(s, blocks, offset):
    """Keys and values of given places, fp32 [nkv, ...places, hd]; negative blocks are read as block 0."""
    c, at = s["case"], blocks.clamp(min=0).long()

    def one(pool, scale):
        x = _values(pool.permute(0, 2, 1, 3)[at, offset], c["fmt"]) * scale[at][..., None]
        return x.movedim(-2, 0)

    return one(s["k"], s["ks"]), one(s["v"], s["vs"])


def _attention(s):
    """Softmax attention over the dequantised tokens: those of the prefix, the same for all, and each
    sequence's own, padded to the most that any of them sees."""
    c = s["case"]
    b, n, group, hd, nkv, bt = c["seqs"], c["new"], c["group"], c["hd"], c["nkv"], c["bt"]
    past = s["lengths"].long()
    most = max(lengths_of(c)) + n
    if c["op"] == "prefix":
        places = torch.arange(most, device=DEV).expand(b, most)
    else:
        span = min(c["window"] + n - 1, most)
        late = past[:, None] + n - span + torch.arange(span, device=DEV)
        places = torch.cat((torch.arange(c["first"], device=DEV).expand(b, -1),
                            torch.where(late >= c["first"], late, torch.full_like(late, 1 << 40))), 1)
    held = places < (past + n)[:, None]
    at = torch.where(held, places, torch.zeros_like(places))
    key, val = _tokens(s, torch.gather(s["table"].long(), 1, at // bt), at % bt)   # [nkv, b, T, hd]
    q = s["q"].float().view(b, n, nkv, group, hd).permute(2, 0, 1, 3, 4).reshape(nkv, b, n * group, hd) / math.sqrt(hd)
    z = torch.matmul(q, key.transpose(2, 3)).view(nkv, b, n, group, -1)
    pos = past[:, None] + torch.arange(n, device=DEV)
    ok = held[:, None] & (places[:, None] <= pos[..., None])
    if c["op"] == "sinks":
        ok &= (places[:, None] < c["first"]) | (places[:, None] > pos[..., None] - c["window"])
    if s["mask"] is not None:
        ok &= (torch.gather(s["mask"], 1, at) != 0)[:, None]
    z = z.masked_fill(~ok[None, :, :, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    if c["op"] == "prefix":
        t = torch.arange(c["pre"], device=DEV)
        pre_key, pre_val = _tokens(s, s["pre"][t // bt], t % bt)                    # [nkv, P, hd]
        pz = torch.matmul(q.reshape(nkv, b * n * group, hd), pre_key.transpose(1, 2)).view(nkv, b, n, group, -1)
        top = torch.maximum(top, pz.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(z - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(nkv, b, n * group, -1), val).view(nkv, b, n, group, hd)
    if c["op"] == "prefix":
        pp = torch.exp(pz - top)
        total = total + pp.sum(-1, keepdim=True)
        o = o + torch.matmul(pp.reshape(nkv, b * n * group, -1), pre_val).view(nkv, b, n, group, hd)
    o = o / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + torch.log(total))[..., 0]
    o = o.permute(1, 2, 0, 3, 4).reshape(b * n, nkv * group, hd)
    return o.to(torch.bfloat16), lse.permute(1, 2, 0, 3).reshape(b * n, nkv * group)


# --------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    global own
    keep, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = keep
    return _exact_w8(s) if case["op"] == "w8" else _exact_attention(s)


def _exact_w8(s):
    """The format's own rule in 64 bits: a token's scale is stored in 32 bits, and a code is the nearest
    to the quotient in 32 bits."""
    x = s["x"].double()
    if s["norm"] is not None:
        x = x / torch.sqrt(x.square().sum(1, keepdim=True) / x.shape[1] + EPS) * s["norm"].double()
    scale = (x.abs().amax(1) / INT8_MAX).float().double()
    quot = torch.nan_to_num((x / scale[:, None]).float().double())
    code = quot.round().clamp(-INT8_MAX, INT8_MAX)
    y = torch.empty(x.shape[0], s["codes"].shape[0], dtype=torch.float64, device=DEV)
    for i in range(0, y.shape[1], 4096):
        w = s["codes"][i:i + 4096].double() * s["scales"][i:i + 4096].double()[:, None]
        y[:, i:i + 4096] = (code @ w.t()) * scale[:, None]
    return y if s["resid"] is None else y + s["resid"].double()


def _exact_attention(s):
    c = s["case"]
    n, group, hd, nkv, bt = c["new"], c["group"], c["hd"], c["nkv"], c["bt"]
    o = torch.zeros(s["rows"], nkv * group, hd, dtype=torch.float64, device=DEV)
    lse = torch.full((s["rows"], nkv * group), -math.inf, dtype=torch.float64, device=DEV)

    def read(ids, within):
        key = _values(s["k"][ids, :, within], c["fmt"]).double() * s["ks"][ids].double()[..., None]
        val = _values(s["v"][ids, :, within], c["fmt"]).double() * s["vs"][ids].double()[..., None]
        return key.transpose(0, 1), val.transpose(0, 1)

    if c["op"] == "prefix":
        t = torch.arange(c["pre"], device=DEV)
        pre_key, pre_val = read(s["pre"].long()[t // bt], t % bt)
    for b, past in enumerate(lengths_of(c)):
        for i in range(n):
            tok = torch.arange(past + i + 1, device=DEV)
            if c["op"] == "sinks":
                tok = tok[(tok < c["first"]) | (past + i - tok < c["window"])]
            if s["mask"] is not None:
                tok = tok[s["mask"][b, tok].bool()]
            key, val = read(s["table"][b].long()[tok // bt], tok % bt)
            if c["op"] == "prefix":
                key, val = torch.cat((pre_key, key), 1), torch.cat((pre_val, val), 1)
            if key.shape[1] == 0:
                continue
            q = s["q"][b * n + i].double().view(nkv, group, hd)
            z = torch.einsum("hgd,htd->hgt", q, key) / math.sqrt(hd)
            one = torch.logsumexp(z, -1)
            o[b * n + i] = torch.einsum("hgt,htd->hgd", torch.exp(z - one[..., None]), val).view(nkv * group, hd)
            lse[b * n + i] = one.view(-1)
    return o, lse
