"""The decoding example (glt_b200.decode): prompt and single tokens through 4-bit projections,
the 8-bit cache, its attention and the token probabilities, step by step against a 32-bit
forward of each step's token over the same (unpacked) weights and the cache's values of that step.

Tolerance: each of the two layers rounds its activations to bf16 about ten times (2^-9 each,
relative): some 2 % of the logits' spread, which is about 1; 0.05 is taken."""
import math

import pytest
import torch

from glt_b200 import decode, serve

pytestmark = pytest.mark.gpu
HID, F, L, NH, NKV, HD, V = 256, 640, 2, 4, 2, 64, 512
THETA = 1e4


def reference(d, ids):
    """fp32 logits [seqs, V] of the last tokens ids [seqs], which the cache holds already, with the
    decoder's own rounded weights."""
    def w(x):
        return x.unpack().float()

    T = int(d.lengths[0])
    x = d.embed[ids].float()
    held = serve.Kv8Batch(d.table, d.lengths, 0, max_new=0)

    def norm(y, g):
        return y * torch.rsqrt(y.square().mean(-1, keepdim=True) + d.eps) * g.float()

    for y in d.layers:
        q = (norm(x, y["in_norm"]) @ w(y["qkv"]).t()).unflatten(-1, (-1, HD))[:, :NH]
        a, b = q.chunk(2, -1)
        c, s = d.cos[T - 1], d.sin[T - 1]
        q = torch.cat((a * c - b * s, a * s + b * c), -1)[:, :, None]
        k, v = (t.transpose(1, 2).repeat_interleave(NH // NKV, 1) for t in y["cache"].read(held, None, T))
        p = torch.softmax(q @ k.transpose(2, 3) / math.sqrt(HD), -1)
        x = x + (p @ v).flatten(1) @ w(y["o"]).t()
        gate, up = (norm(x, y["post_norm"]) @ w(y["gate_up"]).t()).chunk(2, -1)
        x = x + (torch.nn.functional.silu(gate) * up) @ w(y["down"]).t()
    return norm(x, d.final_norm) @ w(d.head).t()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_decoding_matches_each_step(fmt):
    w = decode.random_weights(HID, F, L, NH, NKV, HD, V, seed=3, std=0.06)
    d = decode.Decoder(w, NH, NKV, HD, seqs=3, max_tokens=96, group=32, block_tokens=16, fmt=fmt, rope_theta=THETA)
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, V, (3, 41), device="cuda", dtype=torch.int32, generator=g)
    for _ in range(20):
        logits = d.step(ids)
        want = reference(d, ids[:, -1])
        tol = 0.05 * max(want.std().item(), 1.0)
        assert (logits - want).abs().max().item() < 4 * tol      # the largest of 512 logits
        r = serve.token_logprobs(logits, top=1)
        ref = torch.log_softmax(want, -1)
        got = ref.gather(1, r.top_ids.long())
        assert (got - r.top_logp).abs().max().item() < tol
        assert (ref.amax(-1) - got[:, 0]).max().item() < 2 * tol  # the chosen token is the best one, up to the tolerance
        ids = r.top_ids
    assert d.lengths.tolist() == [41 + 19] * 3


def test_generate_is_step_by_step():
    w = decode.random_weights(HID, F, L, NH, NKV, HD, V, seed=7, std=0.06)
    prompt = torch.randint(0, V, (2, 12), device="cuda", dtype=torch.int32, generator=torch.Generator(device="cuda").manual_seed(2))
    a, b = (decode.Decoder(w, NH, NKV, HD, seqs=2, max_tokens=64, rope_theta=THETA) for _ in range(2))
    ids, logps = a.generate(prompt, 6)
    cur = prompt
    for i in range(6):
        r = serve.token_logprobs(b.step(cur), top=1)
        assert torch.equal(r.top_ids[:, 0], ids[:, i]) and torch.equal(r.top_logp[:, 0], logps[:, i])
        cur = r.top_ids


def test_prompt_in_one_step_or_token_by_token():
    w = decode.random_weights(HID, F, L, NH, NKV, HD, V, seed=4, std=0.06)
    prompt = torch.randint(0, V, (2, 23), device="cuda", dtype=torch.int32, generator=torch.Generator(device="cuda").manual_seed(3))
    out = []
    for cut in ([23], [1] * 23, [5, 17, 1]):
        d = decode.Decoder(w, NH, NKV, HD, seqs=2, max_tokens=64, group=64, block_tokens=32, rope_theta=THETA)
        at = 0
        for n in cut:
            logits = d.step(prompt[:, at:at + n].contiguous())
            at += n
        out.append(logits)
    tol = 0.05 * max(out[0].std().item(), 1.0)
    assert (out[0] - out[1]).abs().max() < 2 * tol and (out[0] - out[2]).abs().max() < 2 * tol


def test_given_tokens_score_like_generated_ones():
    w = decode.random_weights(HID, F, L, NH, NKV, HD, V, seed=5, std=0.06)
    d = decode.Decoder(w, NH, NKV, HD, seqs=2, max_tokens=64, rope_theta=THETA)
    logits = d.step(torch.randint(0, V, (2, 9), device="cuda", dtype=torch.int32))
    r = serve.token_logprobs(logits, top=3)
    s = serve.token_logprobs(logits, r.top_ids[:, 1].contiguous())
    assert torch.equal(s.logp, r.top_logp[:, 1])
