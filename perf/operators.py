"""Cases that measure the decoding and scoring operators, with their plain forms.

Three operators: attention over an 8-bit key/value cache (and the append that fills it),
products with 4-bit weights, and log probabilities of given tokens with entropy, alternatives
and gradient.  ``own`` selects what ``run`` computes with: elementary torch operations in
32 bits, or the library's entry points in ``glt_b200.serve``.
"""
import math
import random

import torch

own = False

DEV = "cuda"
INT8_MAX, E4M3_MAX = 127.0, 448.0


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one user's next token on the Qwen2.5-0.5B head layout: launch latency counts
        attn("attend_one_user", fmt="int8", bt=16, seqs=1, ctx=1001, nkv=2, group=7, hd=64),
        # a serving batch on the Llama-3-8B head layout, users at very different positions
        attn("attend_batch", fmt="int8", bt=64, seqs=32, ctx=8191, ragged=True, nkv=8, group=4, hd=128),
        # a few long documents, one token at a time
        attn("attend_long", fmt="e4m3", bt=128, seqs=4, ctx=65537, nkv=8, group=4, hd=128),
        # five draft tokens a user, checked at once, with a sliding window and dropped tokens
        attn("attend_drafts", fmt="e4m3", bt=32, seqs=12, ctx=5003, ragged=True, new=5, nkv=4, group=8,
             hd=128, window=4095, masked=True),
        # every user's new token goes into a block that already holds some
        append("append_step", fmt="int8", bt=16, seqs=64, ctx=777, ragged=True, new=1, nkv=8, hd=128),
        # prompts of different lengths enter the cache
        append("append_prompts", fmt="e4m3", bt=64, seqs=6, ctx=130, ragged=True, new=2047, nkv=8, hd=128),
        # single token through the Qwen2.5-0.5B down projection
        w4("w4_small", m=1, n=896, k=4864, g=128),
        # single token through the Llama-3-8B gate and up projections
        w4("w4_gate_up", m=1, n=28672, k=4096, g=128),
        # a batch through the Llama-3-8B down projection, finer groups with zero points, residual
        w4("w4_down_batch", m=19, n=4096, k=14336, g=32, asym=True, resid=True),
        # sampling: a few rows of Qwen2.5-0.5B logits, part of the vocabulary forbidden
        logp("logp_sample", rows=5, v=151936, top=20, scale=1.25, masked=True),
        # scoring: rows of Llama-3-8B logits with a few alternatives
        logp("logp_score", rows=4096, v=128256, top=5),
        # policy training: forward and gradient, odd vocabulary
        logp("logp_train", rows=2047, v=128257, top=0, train=True),
    ]


def attn(name, **kw):
    return dict(dict(name=name, op="attention", ragged=False, new=1, window=0, masked=False), **kw)


def append(name, **kw):
    return dict(dict(name=name, op="append", ragged=False), **kw)


def w4(name, **kw):
    return dict(dict(name=name, op="w4", asym=False, resid=False, out="bf16"), **kw)


def logp(name, **kw):
    return dict(dict(name=name, op="logp", scale=1.0, masked=False, train=False, dtype="bf16"), **kw)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _odd(rng, lo, hi):
    return 2 * (_log(rng, lo, hi) // 2) + 1


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "w4", "w4", "logp", "logp"])
    if op in ("attention", "append"):
        hd, nkv = rng.choice([64, 128]), rng.choice([1, 2, 4, 8])
        fmt, bt = rng.choice(["int8", "e4m3"]), rng.choice([16, 32, 64, 128])
        seqs = _log(rng, 1, 64)
        if op == "append":
            new = _log(rng, 1, max(1, min(2047, 12000 // seqs)))
            c = append("", fmt=fmt, bt=bt, seqs=seqs, ctx=_log(rng, 1, 1000), ragged=rng.random() < 0.5,
                       new=new, nkv=nkv, hd=hd)
        else:
            new = rng.choice([1, 1, 1, 2, 3, 4, 7])
            top = min(65537, 4 * 65537 * 8 * 128 // (seqs * nkv * hd * new))
            c = attn("", fmt=fmt, bt=bt, seqs=seqs, ctx=_odd(rng, 1, top - 1), ragged=rng.random() < 0.5,
                     new=new, nkv=nkv, group=rng.choice([1, 2, 3, 4, 6, 7, 8]), hd=hd,
                     window=rng.choice([0, 0, _odd(rng, 1, 8191)]), masked=rng.random() < 0.3)
    elif op == "w4":
        g = rng.choice([32, 64, 128])
        c = w4("", m=_log(rng, 1, 32), n=_odd(rng, 64, 28671), k=g * _odd(rng, max(1, 512 // g), 14335 // g),
               g=g, asym=rng.random() < 0.5, resid=rng.random() < 0.5, out=rng.choice(["bf16", "fp32"]))
        while c["n"] * c["k"] > 28672 * 4096:
            c["n"] = 2 * (c["n"] // 4) + 1
    else:
        v = _odd(rng, 1001, 151935)
        dtype, train = rng.choice(["bf16", "bf16", "fp32"]), rng.random() < 0.4
        rows = _odd(rng, 1, max(2, min(4095, 2047 * 128257 // (v * (2 if dtype == "fp32" else 1)))))
        c = logp("", rows=rows, v=v, top=rng.choice([0, 1, 4, 5]) if rows > 64 else rng.choice([0, 1, 5, 20, 32]),
                 scale=rng.choice([1.0, 0.7, 1.6]), masked=rng.random() < 0.3, train=train, dtype=dtype)
    del c["name"]
    return c


# --------------------------------------------------------------------------- sizes
def lengths_of(c):
    """Tokens in the cache before the call: ctx for all, or spread from nearly none to ctx."""
    n = c["seqs"]
    if not c["ragged"]:
        return [c["ctx"]] * n
    r = random.Random(n * 1000003 + c["ctx"])
    return [c["ctx"] if i == 0 else int(c["ctx"] * r.random() ** 1.5) for i in range(n)]


def news_of(c):
    """New tokens of each sequence (ragged prompts: from one to all of them)."""
    if c["op"] == "append" and c["ragged"] and c["new"] > 1:
        r = random.Random(c["new"])
        return [c["new"] if i == 0 else r.randint(1, c["new"]) for i in range(c["seqs"])]
    return [c["new"]] * c["seqs"]


def _blocks(c):
    """Blocks held by each sequence after the call."""
    return [-(-(a + b) // c["bt"]) for a, b in zip(lengths_of(c), news_of(c))]


def _span(c):
    """Most blocks any one sequence's new tokens reach into."""
    return max((a + b - 1) // c["bt"] - a // c["bt"] + 1 for a, b in zip(lengths_of(c), news_of(c)))


def work(c):
    if c["op"] == "attention":
        per, hd, nh = c["nkv"] * c["hd"], c["hd"], c["nkv"] * c["group"]
        seen = pairs = 0
        for past in lengths_of(c):
            first = max(0, past + 1 - c["window"]) if c["window"] else 0
            seen += past + c["new"] - first
            for i in range(c["new"]):
                end = past + i + 1
                pairs += min(end, c["window"]) if c["window"] else end
        rows = c["seqs"] * c["new"]
        byt = 2 * seen * per + 8 * c["nkv"] * (seen // c["bt"] + c["seqs"]) + 4 * rows * nh * hd + 4 * rows * nh
        if c["masked"]:
            byt += seen
        return {"bytes": byt, "flops": 4 * pairs * nh * hd}
    if c["op"] == "append":
        rows, per = sum(news_of(c)), c["nkv"] * c["hd"]
        vals = c["seqs"] * _span(c) * c["bt"] * per
        return {"bytes": 4 * rows * per + 2 * rows * per + 8 * vals, "flops": 6 * rows * per}
    if c["op"] == "w4":
        m, n, k, g = c["m"], c["n"], c["k"], c["g"]
        byt = n * k // 2 + n * (k // g) * (3 if c["asym"] else 2) + 2 * m * k + m * n * (2 if c["out"] == "bf16" else 4)
        return {"bytes": byt + (2 * m * n if c["resid"] else 0), "flops": 2 * m * n * k}
    es = 2 if c["dtype"] == "bf16" else 4
    one = c["rows"] * c["v"]
    return {"bytes": one * es * (2 if c["train"] else 1), "flops": one * (12 if c["train"] else 6)}


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _quant(x, s, fmt):
    """8-bit codes (uint8) of x / s: int8 stored with an offset of 128, or e4m3."""
    y = torch.where(s > 0, x / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(x))
    if fmt == "int8":
        return (y.round().clamp(-127, 127) + 128).to(torch.uint8)
    return y.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)


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
        pool[i:i + 1024] = _quant(x, s, fmt)
        scale[i:i + 1024] = s[:, :, 0, 0]


def _prepare_cache(c, seed):
    g = _gen(seed)
    held = _blocks(c)
    nb, maxb = sum(held) + 3, max(held)
    perm = torch.randperm(nb, device=DEV, generator=g).to(torch.int32)
    table = torch.zeros(c["seqs"], maxb, dtype=torch.int32, device=DEV)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = perm[at:at + h]
        at += h
    shape = (nb, c["nkv"], c["bt"], c["hd"])
    k, v = (torch.empty(shape, dtype=torch.uint8, device=DEV) for _ in range(2))
    ks, vs = (torch.empty(nb, c["nkv"], device=DEV) for _ in range(2))
    _fill(k, ks, g, c["fmt"], "k")
    _fill(v, vs, g, c["fmt"], "v")
    lens, news = lengths_of(c), news_of(c)
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    s = dict(case=c, k=k, v=v, ks=ks, vs=vs, table=table, rows=starts[-1],
             lengths=torch.tensor(lens, dtype=torch.int32, device=DEV),
             row_start=torch.tensor(starts, dtype=torch.int32, device=DEV),
             even=len(set(news)) == 1, max_new=max(news))
    if c["op"] == "attention":
        nh = c["nkv"] * c["group"]
        # a packed row as the query/key/value projection leaves it: the queries are its first columns
        qkv = torch.randn(s["rows"], (nh + 2 * c["nkv"]) * c["hd"], device=DEV, generator=g).to(torch.bfloat16)
        s["q"] = qkv[:, :nh * c["hd"]].view(s["rows"], nh, c["hd"])
        s["mask"] = None
        if c["masked"]:
            keep = torch.rand(c["seqs"], maxb * c["bt"], device=DEV, generator=g) > 0.25
            s["mask"] = keep.to(torch.uint8)
    else:
        kv = torch.randn(s["rows"], 2, c["nkv"], c["hd"], device=DEV, generator=g) * 1.5
        kv = kv.to(torch.bfloat16)
        s["new_k"], s["new_v"] = kv[:, 0], kv[:, 1]
        s["start"] = s["lengths"] // c["bt"] * c["bt"]
        s["count"] = _span(c) * c["bt"]
    if own:
        from glt_b200 import serve
        s["cache"] = serve.Kv8Cache.from_buffers(k, v, ks, vs, c["fmt"])
        s["batch"] = serve.Kv8Batch(table, s["lengths"], s["rows"],
                                    row_start=None if s["even"] else s["row_start"], max_new=s["max_new"])
    return s


def _prepare_w4(c, seed):
    g = _gen(seed)
    m, n, k, grp = c["m"], c["n"], c["k"], c["g"]
    w = (torch.randn(n, k, device=DEV, generator=g) * 0.02).view(n, k // grp, grp)
    if c["asym"]:
        lo, hi = w.amin(-1, keepdim=True).clamp(max=0), w.amax(-1, keepdim=True).clamp(min=0)
        scale = ((hi - lo) / 15).to(torch.bfloat16)
        zero = (-lo / scale.float()).round().clamp(0, 15)
    else:
        scale = (w.abs().amax(-1, keepdim=True) / 7).to(torch.bfloat16)
        zero = torch.full_like(scale, 8.0, dtype=torch.float32)
    codes = ((w / scale.float()).round() + zero).clamp(0, 15).to(torch.uint8).view(n, k)
    s = dict(case=c, x=torch.randn(m, k, device=DEV, generator=g).to(torch.bfloat16), codes=codes,
             scale=scale.view(n, k // grp), zero=zero.view(n, k // grp).to(torch.uint8), resid=None)
    if c["resid"]:
        s["resid"] = torch.randn(m, n, device=DEV, generator=g).to(torch.bfloat16)
    if own:
        from glt_b200 import serve
        s["weight"] = serve.W4Weight.from_codes(codes, s["scale"], s["zero"] if c["asym"] else None)
        del s["codes"], s["scale"], s["zero"]
    else:
        # two codes a byte, as the checkpoint of such a model stores them
        pad = codes.view(n, k // 2, 2)
        s["codes"] = pad[:, :, 0] | (pad[:, :, 1] << 4)
    return s


def _prepare_logp(c, seed):
    g = _gen(seed)
    dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
    rows, v = c["rows"], c["v"]
    x = torch.empty(rows, v, device=DEV, dtype=dt)
    t = torch.randint(0, v, (rows,), device=DEV, generator=g)
    for i in range(0, rows, 512):
        y = torch.randn(min(512, rows - i), v, device=DEV, generator=g) * 2.5
        # a handful of likely tokens a row, the given one often among them
        hot = torch.randint(0, v, (y.shape[0], 12), device=DEV, generator=g)
        hot[::2, 0] = t[i:i + 512][::2]
        y.scatter_add_(1, hot, torch.rand(hot.shape, device=DEV, generator=g) * 14)
        if c["masked"]:
            # a grammar forbids part of the vocabulary, never the given token
            keep = y.gather(1, t[i:i + 512, None])
            y[:, torch.rand(v, device=DEV, generator=g) < 0.4] = -math.inf
            y.scatter_(1, t[i:i + 512, None], keep)
        x[i:i + 512] = y
    t[::7] = -1  # positions without a given token
    s = dict(case=c, x=x, t=t.to(torch.int32))
    if c["train"]:
        s["d_logp"] = torch.randn(rows, device=DEV, generator=g)
        s["d_entropy"] = torch.randn(rows, device=DEV, generator=g) * 0.1
    return s


def prepare(case, seed):
    if case["op"] in ("attention", "append"):
        return _prepare_cache(case, seed)
    return (_prepare_w4 if case["op"] == "w4" else _prepare_logp)(case, seed)


# --------------------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return {"attention": _own_attention, "append": _own_append, "w4": _own_w4, "logp": _own_logp}[op](s)
    if op == "attention":
        return _attention(s, torch.float32)
    if op == "append":
        return _append(s)
    if op == "w4":
        return _w4(s)
    return _logp(s)


def _own_attention(s):
    return s["cache"].attention(s["batch"], s["q"], window=s["case"]["window"], token_mask=s["mask"])


def _own_append(s):
    s["cache"].append(s["batch"], s["new_k"], s["new_v"])
    return s["cache"].read(s["batch"], s["start"], s["count"])


def _own_w4(s):
    return s["weight"].linear(s["x"], resid=s["resid"],
                              out_dtype=torch.bfloat16 if s["case"]["out"] == "bf16" else torch.float32)


def _own_logp(s):
    from glt_b200 import serve
    c = s["case"]
    r = serve.token_logprobs(s["x"], s["t"], scale=c["scale"], top=c["top"])
    out = [r.logp, r.entropy, r.lse]
    if c["top"]:
        out += [r.top_ids, r.top_logp]
    if c["train"]:
        out.append(serve.token_logprobs_bwd(s["x"], s["t"], r, s["d_logp"], s["d_entropy"]))
    return out


def _attention(s, dt, seqs=None):
    """Softmax attention over the dequantised cache, all sequences padded to the longest
    (``seqs``: only those).  Every sequence has the same number of new tokens."""
    c = s["case"]
    n, group, hd, nkv, bt = c["new"], c["group"], c["hd"], c["nkv"], c["bt"]
    sel = slice(None) if seqs is None else seqs
    table, past = s["table"][sel].long(), s["lengths"][sel].long()
    b, maxb = table.shape
    ctx = maxb * bt

    def gather(pool, scale):
        x = _values(pool[table], c["fmt"]).to(dt) * scale[table].to(dt)[..., None, None]
        return x.transpose(1, 2).reshape(b, nkv, ctx, hd)

    q = s["q"].view(c["seqs"], n, nkv, group, hd)[sel].to(dt)
    q = q.permute(0, 2, 3, 1, 4).reshape(b, nkv, group * n, hd) * (1.0 / math.sqrt(hd))
    z = torch.matmul(q, gather(s["k"], s["ks"]).transpose(2, 3)).view(b, nkv, group, n, ctx)
    pos = past[:, None] + torch.arange(n, device=DEV)
    t = torch.arange(ctx, device=DEV)
    ok = t <= pos[..., None]
    if c["window"]:
        ok &= t > pos[..., None] - c["window"]
    if s["mask"] is not None:
        ok &= (s["mask"][sel] != 0)[:, None, :]
    z = z.masked_fill(~ok[:, None, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(z - top)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(p.view(b, nkv, group * n, ctx), gather(s["v"], s["vs"])).view(b, nkv, group, n, hd)
    lse = (top + torch.log(total))[..., 0]
    o = o.permute(0, 3, 1, 2, 4).reshape(b * n, nkv * group, hd)
    lse = lse.permute(0, 3, 1, 2).reshape(b * n, nkv * group)
    return (o.to(torch.bfloat16), lse) if dt == torch.float32 else (o, lse)


def _append(s):
    """Quantises the new rows into their blocks; returns the values of all blocks written to."""
    c = s["case"]
    b, bt, nkv, hd, fmt = c["seqs"], c["bt"], c["nkv"], c["hd"], c["fmt"]
    span = s["count"] // bt
    lo = s["row_start"][:-1].long()
    new = s["row_start"][1:].long() - lo
    past = s["lengths"].long()
    pos = s["start"].long()[:, None] + torch.arange(s["count"], device=DEV)
    row = (lo[:, None] + pos - past[:, None]).clamp(0, s["rows"] - 1)
    fresh = (pos >= past[:, None]) & (pos < (past + new)[:, None])
    held = pos < past[:, None]
    at = (pos[:, ::bt] // bt).clamp(max=s["table"].shape[1] - 1)
    touched = pos[:, ::bt] < (past + new)[:, None]
    blocks = torch.gather(s["table"].long(), 1, at)

    def one(pool, scale, x):
        old = pool[blocks].transpose(2, 3).reshape(b, s["count"], nkv, hd)
        some = held.view(b, span, bt)[:, :, 0][..., None]
        before = torch.where(some, scale[blocks], torch.zeros_like(scale[blocks]))
        wide = before.repeat_interleave(bt, 1)[..., None]
        vals = torch.where(held[..., None, None], _values(old, fmt) * wide, torch.zeros_like(wide))
        incoming = torch.where(fresh[..., None, None], x[row].float(), torch.zeros_like(wide))
        peak = incoming.abs().view(b, span, bt, nkv, hd).amax((2, 4))
        # a tensor divisor: a plain number would become a product with its rounded reciprocal
        after = torch.maximum(before, peak / torch.full_like(peak, INT8_MAX if fmt == "int8" else E4M3_MAX))
        wide = after.repeat_interleave(bt, 1)[..., None]
        codes = _quant(torch.where(fresh[..., None, None], incoming, vals), wide, fmt)
        keep = touched[..., None, None, None]
        codes_b = codes.view(b, span, bt, nkv, hd).transpose(2, 3)
        dst = blocks[touched]
        pool[dst] = codes_b[touched]
        scale[dst] = after[touched]
        out = _values(codes, fmt) * wide
        live = (fresh | held)[..., None, None] & keep.repeat_interleave(bt, 1)[..., 0]
        return torch.where(live, out, torch.zeros_like(out))

    return one(s["k"], s["ks"], s["new_k"]), one(s["v"], s["vs"], s["new_v"])


def _w4(s):
    c = s["case"]
    n, k, g = c["n"], c["k"], c["g"]
    u = torch.stack((s["codes"] & 15, s["codes"] >> 4), -1).view(n, k // g, g).float()
    w = ((u - s["zero"].float()[..., None]) * s["scale"].float()[..., None]).view(n, k)
    y = torch.matmul(s["x"].float(), w.t())
    if s["resid"] is not None:
        y = y + s["resid"].float()
    return y.to(torch.bfloat16) if c["out"] == "bf16" else y


def _logp(s):
    c = s["case"]
    x, t = s["x"].float(), s["t"].long()
    given = t >= 0
    z = x * c["scale"]
    top = z.amax(-1, keepdim=True)
    lse = (top + torch.log(torch.exp(z - top).sum(-1, keepdim=True)))
    p = torch.exp(z - lse)
    ent = lse[:, 0] - torch.where(p > 0, p * z, torch.zeros_like(p)).sum(-1)
    zt = torch.gather(z, 1, t.clamp(min=0)[:, None])[:, 0]
    lp = torch.where(given, zt - lse[:, 0], torch.zeros_like(zt))
    out = [lp, ent, lse[:, 0]]
    if c["top"]:
        iota = torch.arange(c["v"], device=DEV, dtype=torch.int32)
        left, ids = x.clone(), []
        taken = torch.zeros_like(x, dtype=torch.bool)
        for _ in range(c["top"]):
            best = left.amax(-1, keepdim=True)
            # the lowest index among equals that is not taken yet
            i = torch.where((left == best) & ~taken, iota, c["v"]).amin(-1, keepdim=True)
            ids.append(i)
            left.scatter_(1, i.long(), -math.inf)
            taken.scatter_(1, i.long(), True)
        ids = torch.cat(ids, 1)
        out += [ids, torch.gather(z, 1, ids.long()) - lse]
    if c["train"]:
        dl = torch.where(given, s["d_logp"], torch.zeros_like(lp))[:, None]
        de = s["d_entropy"][:, None]
        spread = torch.where(p > 0, z - lse + ent[:, None], torch.zeros_like(p))
        dz = -p * (dl + de * spread)
        dz.scatter_add_(1, t.clamp(min=0)[:, None], dl)
        out.append((dz * c["scale"]).to(s["x"].dtype))
    return out


# --------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    global own
    keep, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = keep
    return {"attention": _exact_attention, "append": _exact_append, "w4": _exact_w4, "logp": _exact_logp}[case["op"]](s)


def _exact_attention(s):
    c = s["case"]
    n, group, hd, nkv, bt = c["new"], c["group"], c["hd"], c["nkv"], c["bt"]
    o = torch.zeros(s["rows"], nkv * group, hd, dtype=torch.float64, device=DEV)
    lse = torch.full((s["rows"], nkv * group), -math.inf, dtype=torch.float64, device=DEV)
    for b, past in enumerate(lengths_of(c)):
        ids = s["table"][b, :-(-(past + n) // bt)].long()
        tok = torch.arange(past + n, device=DEV)
        for h in range(nkv):
            key = (_values(s["k"][ids, h], c["fmt"]).double() * s["ks"][ids, h].double()[:, None, None]).view(-1, hd)
            val = (_values(s["v"][ids, h], c["fmt"]).double() * s["vs"][ids, h].double()[:, None, None]).view(-1, hd)
            for i in range(n):
                see = tok <= past + i
                if c["window"]:
                    see = see & (past + i - tok < c["window"])
                if s["mask"] is not None:
                    see = see & s["mask"][b, :past + n].bool()
                see = see.nonzero()[:, 0]
                if not see.numel():
                    continue
                q = s["q"][b * n + i, h * group:(h + 1) * group].double()
                z = (key[see] @ q.t()) / math.sqrt(hd)
                one = torch.logsumexp(z, 0)
                o[b * n + i, h * group:(h + 1) * group] = torch.exp(z - one).t() @ val[see]
                lse[b * n + i, h * group:(h + 1) * group] = one
    return o, lse


def _exact_append(s):
    """The format's own rule in 64 bits: a block's scale is stored in 32 bits, and a code is the
    nearest to the quotient in 32 bits (a 64-bit quotient rounded once more gives that quotient)."""
    c = s["case"]
    bt, fmt = c["bt"], c["fmt"]
    outs = []
    for pool, scale, x in ((s["k"], s["ks"], s["new_k"]), (s["v"], s["vs"], s["new_v"])):
        out = torch.zeros(c["seqs"], s["count"], c["nkv"], c["hd"], dtype=torch.float64, device=DEV)
        at = 0
        for b, (past, new) in enumerate(zip(lengths_of(c), news_of(c))):
            base = past // bt * bt
            for blk in range(past // bt, (past + new - 1) // bt + 1):
                lo, hi = max(past, blk * bt), min(past + new, (blk + 1) * bt)
                rows = x[at + lo - past:at + hi - past].double()
                peak = (rows.abs().amax((0, 2)) / (INT8_MAX if fmt == "int8" else E4M3_MAX)).float().double()
                if lo > blk * bt:
                    i = int(s["table"][b, blk])
                    before = scale[i].double()
                    old = _values(pool[i, :, :lo - blk * bt], fmt).double().transpose(0, 1) * before[:, None]
                    peak = torch.maximum(peak, before)
                    rows = torch.cat((old.float().double(), rows))
                quot = torch.nan_to_num((rows / peak[:, None]).float().double())
                if fmt == "int8":
                    code = quot.round().clamp(-INT8_MAX, INT8_MAX)
                else:
                    code = quot.float().clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).double()
                first = blk * bt - base
                out[b, first:first + rows.shape[0]] = code * peak[:, None]
            at += new
        outs.append(out)
    return tuple(outs)


def _exact_w4(s):
    c = s["case"]
    n, k, g = c["n"], c["k"], c["g"]
    x = s["x"].double()
    y = torch.empty(c["m"], n, dtype=torch.float64, device=DEV)
    for i in range(0, n, 2048):
        two = s["codes"][i:i + 2048].long()
        u = torch.empty(two.shape[0], k, dtype=torch.float64, device=DEV)
        u[:, 0::2], u[:, 1::2] = (two % 16).double(), (two // 16).double()
        u = u.view(-1, k // g, g)
        w = (u - s["zero"][i:i + 2048].double().unsqueeze(-1)) * s["scale"][i:i + 2048].double().unsqueeze(-1)
        y[:, i:i + 2048] = x @ w.reshape(-1, k).t()
    return y if s["resid"] is None else y + s["resid"].double()


def _exact_logp(s):
    c = s["case"]
    parts = []
    for i in range(0, c["rows"], 256):
        raw, t = s["x"][i:i + 256].double(), s["t"][i:i + 256].long()
        logq = torch.log_softmax(raw * c["scale"], -1)
        q = logq.exp()
        lse = torch.logsumexp(raw * c["scale"], -1)
        ent = -torch.nansum(q * logq, -1)  # 0 * -inf, a token that cannot occur, counts nothing
        here = (t >= 0).double()
        pick = logq.gather(1, t.clamp(min=0)[:, None])[:, 0]
        out = [torch.where(t >= 0, pick, torch.zeros_like(pick)), ent, lse]
        if c["top"]:
            ids = torch.sort(raw, dim=-1, descending=True, stable=True).indices[:, :c["top"]]
            out += [ids.to(torch.int32), logq.gather(1, ids)]
        if c["train"]:
            dl, de = s["d_logp"][i:i + 256].double() * here, s["d_entropy"][i:i + 256].double()
            hot = torch.zeros_like(q).scatter_(1, t.clamp(min=0)[:, None], here[:, None])
            dz = dl[:, None] * (hot - q) - de[:, None] * torch.nan_to_num(q * (logq + ent[:, None]), nan=0.0)
            out.append(dz * c["scale"])
        parts.append(out)
    return [torch.cat(p) for p in zip(*parts)]
