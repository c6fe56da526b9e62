"""The decoder with 8-bit projections, a shared prompt, and a window with first tokens: the operators run together, each step
against a 32-bit forward of its token over the decoder's own rounded weights and the cache's values.

Tolerance as in test_gpu_decode: some 2 % of the logits' spread; an activation of 8 bits is off by half a step, 1 / 254 of
its row's largest value, at most 1/2 % of the sum's spread more for each of the eight products: 5 % holds both, and the
largest of 512 logits may be off by four times that."""
import math

import pytest
import torch

from glt_b200 import decode, serve

pytestmark = pytest.mark.gpu
HID, F, L, NH, NKV, HD, V = 256, 640, 2, 4, 2, 64, 512
THETA = 1e4


def matrix(w):
    return w.codes.float() * w.scales[:, None] if isinstance(w, serve.W8Weight) else w.unpack().float()


def reference(d, ids):
    """fp32 logits [seqs, V] of the last tokens ids [seqs], which the cache holds already."""
    T, P = int(d.lengths[0]), int(d.shared_length)
    x = d.embed[ids].float()
    held = serve.Kv8Batch(d.table, d.lengths, 0, max_new=0)

    def norm(y, g):
        return y * torch.rsqrt(y.square().mean(-1, keepdim=True) + d.eps) * g.float()

    t = torch.arange(T, device="cuda")
    see = (t < d.sinks) | (t > T - 1 - d.window) if d.window else t >= 0
    for y in d.layers:
        q = (norm(x, y["in_norm"]) @ matrix(y["qkv"]).t()).unflatten(-1, (-1, HD))[:, :NH]
        a, b = q.chunk(2, -1)
        c, s = d.cos[P + T - 1], d.sin[P + T - 1]
        q = torch.cat((a * c - b * s, a * s + b * c), -1)[:, :, None]
        kv = [k[:, see] for k in y["cache"].read(held, None, T)]
        if P:
            pre = y["cache"].read(serve.Kv8Batch(d.shared_blocks[None], d.shared_length, 0, max_new=0), None, P)
            kv = [torch.cat((p.expand(d.seqs, -1, -1, -1), k), 1) for p, k in zip(pre, kv)]
        k, v = (k.transpose(1, 2).repeat_interleave(NH // NKV, 1) for k in kv)
        p = torch.softmax(q @ k.transpose(2, 3) / math.sqrt(HD), -1)
        x = x + (p @ v).flatten(1) @ matrix(y["o"]).t()
        gate, up = (norm(x, y["post_norm"]) @ matrix(y["gate_up"]).t()).chunk(2, -1)
        x = x + (torch.nn.functional.silu(gate) * up) @ matrix(y["down"]).t()
    return norm(x, d.final_norm) @ matrix(d.head).t()


def ids_of(seed, *shape):
    return torch.randint(0, V, shape, device="cuda", dtype=torch.int32, generator=torch.Generator(device="cuda").manual_seed(seed))


@pytest.mark.parametrize("bits,shared,window,sinks,fmt", [(8, 0, 0, 0, "int8"), (8, 150, 0, 0, "e4m3"), (4, 77, 0, 0, "int8"),
                                                         (8, 0, 24, 3, "int8"), (4, 0, 17, 20, "e4m3")])
def test_each_step(bits, shared, window, sinks, fmt):
    w = decode.random_weights(HID, F, L, NH, NKV, HD, V, seed=3, std=0.06)
    d = decode.Decoder(w, NH, NKV, HD, seqs=3, max_tokens=96, group=32, block_tokens=16, fmt=fmt, rope_theta=THETA, bits=bits,
                       shared_tokens=shared, window=window, sinks=sinks)
    if shared:
        d.share(ids_of(8, shared - 7))
    ids = ids_of(1, 3, 41)
    for _ in range(20):
        logits = d.step(ids)
        want = reference(d, ids[:, -1])
        tol = 0.05 * max(want.std().item(), 1.0)
        assert (logits - want).abs().max().item() < 4 * tol
        ids = serve.token_logprobs(logits, top=1).top_ids
    assert d.lengths.tolist() == [60] * 3 and d.held == 60


@pytest.mark.parametrize("bits", [4, 8])
def test_a_shared_prompt_is_each_sequences_own(bits):
    """Behind a prefix of whole blocks the cache holds the same codes, so the logits agree to the tolerance of two runs."""
    w = decode.random_weights(HID, F, L, NH, NKV, HD, V, seed=4, std=0.06)
    common, rest = ids_of(5, 64), ids_of(6, 2, 9)
    a = decode.Decoder(w, NH, NKV, HD, seqs=2, max_tokens=40, block_tokens=32, rope_theta=THETA, bits=bits, shared_tokens=70)
    b = decode.Decoder(w, NH, NKV, HD, seqs=2, max_tokens=110, block_tokens=32, rope_theta=THETA, bits=bits)
    a.share(common)
    x, y = a.step(rest), b.step(torch.cat((common.expand(2, -1), rest), 1))
    tol = 0.05 * max(y.std().item(), 1.0)
    assert (x - y).abs().max() < 2 * tol
    # another prompt takes its place, and the first again gives the first's logits
    a.reset()
    a.share(ids_of(7, 70))
    other = a.step(rest)
    assert (other - x).abs().max() > 4 * tol
    a.reset()
    a.share(common)
    assert torch.equal(a.step(rest), x)


def test_a_window_that_holds_all_changes_nothing():
    w = decode.random_weights(HID, F, L, NH, NKV, HD, V, seed=5, std=0.06)
    ids = ids_of(2, 2, 30)
    a, b = (decode.Decoder(w, NH, NKV, HD, seqs=2, max_tokens=64, rope_theta=THETA, **kw) for kw in ({}, dict(window=64, sinks=2)))
    assert torch.equal(a.step(ids), b.step(ids))


def test_the_command_runs(monkeypatch, capsys):
    small = decode.random_weights(HID, F, L, NH, NKV, HD, 1024, seed=1)
    monkeypatch.setattr(decode, "random_weights", lambda **k: small)
    real = decode.Decoder
    monkeypatch.setattr(decode, "Decoder", lambda w, **k: real(w, **{**k, "heads": NH, "kv_heads": NKV, "head_dim": HD}))
    real_randint = torch.randint
    monkeypatch.setattr(torch, "randint", lambda lo, hi, *a, **k: real_randint(lo, 1024, *a, **k))
    for args in (["--bits", "8", "--shared", "50"], ["--window", "12", "--sinks", "2"]):
        monkeypatch.setattr("sys.argv", ["decode", "--seqs", "2", "--prompt", "9", "--tokens", "5"] + args)
        decode.main()
        assert "tokens/s" in capsys.readouterr().out
