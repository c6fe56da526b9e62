"""Greedy decoding of a decoder whose projections are in 4 bits or 8 and whose key/value cache is in 8,
built from the operators of ``glt_b200.serve`` and the layer kernels of the C ABI.

``Decoder`` takes the (baked) bf16 weights of a model, rounds its projections to 4 bits and keeps a
cache for a batch of sequences; ``step`` runs any number of new tokens of each sequence (a
prompt or one token) and returns the logits of the last one; ``generate`` decodes and returns
the tokens with their log probabilities.  ``share`` runs a prompt that all sequences begin with once,
for all of them; with a window, old tokens but a few first ones drop out of sight (the cache holds
``max_tokens`` all the same).

Usage:  python -m glt_b200.decode [--seqs N] [--prompt N] [--tokens N] [--bits 4|8] [--shared N] [--window N --sinks N]
(random weights of the Qwen2.5-0.5B shape; prints tokens per second)
"""
from __future__ import annotations

import argparse
import ctypes as C
import time

import torch

from . import serve
from ._lib import check, lib


def _p(t: torch.Tensor) -> C.c_void_p:
    return C.c_void_p(t.data_ptr())


def random_weights(hidden, intermediate, layers, heads, kv_heads, head_dim, vocab, seed=0, std=0.02, device="cuda"):
    """Random bf16 weights under the names ``Decoder`` reads (HF shapes)."""
    g = torch.Generator(device=device).manual_seed(seed)

    def rn(*shape):
        return (torch.randn(*shape, device=device, generator=g) * std).to(torch.bfloat16)

    def ones():
        return torch.ones(hidden, dtype=torch.bfloat16, device=device)

    per_layer = [dict(in_norm=ones(), q=rn(heads * head_dim, hidden), k=rn(kv_heads * head_dim, hidden),
                      v=rn(kv_heads * head_dim, hidden), o=rn(hidden, heads * head_dim), post_norm=ones(),
                      gate=rn(intermediate, hidden), up=rn(intermediate, hidden), down=rn(hidden, intermediate))
                 for _ in range(layers)]
    return dict(embed=rn(vocab, hidden), final_norm=ones(), layers=per_layer)


class Decoder:
    """A decoder over projections of 4 or 8 ``bits`` (the head is the embedding's transpose) and an 8-bit cache.

    The cache holds ``seqs`` sequences of up to ``max_tokens`` tokens behind a shared prefix of up to
    ``shared_tokens``; ``lengths`` counts the tokens each one has on the device, ``held`` on the host, neither the
    prefix's.  ``reset`` forgets the sequences.  With ``window``, a token sees the last ``window`` tokens and the first
    ``sinks`` (no prefix then).

    A sequence that was given an id outside the vocabulary gets logits of NaN from then on, until ``reset``, and all of
    them do behind a shared prefix with one: the host does not wait to look at the ids, and the cache holds nothing
    right of such a token."""

    prefix = unknown = None
    window = sinks = 0

    def __init__(self, weights: dict, heads: int, kv_heads: int, head_dim: int, seqs: int, max_tokens: int,
                 group: int = 64, block_tokens: int = 64, fmt: str = "int8", rope_theta: float = 1e6,
                 eps: float = 1e-6, bits: int = 4, shared_tokens: int = 0, window: int = 0, sinks: int = 0):
        if bits not in (4, 8):
            raise ValueError(f"projections of {bits} bits (4 or 8)")
        if shared_tokens < 0 or window < 0 or sinks < 0 or (window and shared_tokens) or (sinks and not window):
            raise ValueError("shared_tokens, window and sinks must not be negative; a window excludes a shared prefix, "
                             "and sinks need a window")
        self.window, self.sinks = window, sinks
        self.heads, self.kv_heads, self.head_dim, self.seqs, self.eps = heads, kv_heads, head_dim, seqs, eps
        self.max_tokens, self.held = max_tokens, 0
        self.embed, self.final_norm = weights["embed"], weights["final_norm"]
        dev = self.embed.device

        def quantize(matrix):
            return serve.W8Weight.quantize(matrix) if bits == 8 else serve.W4Weight.quantize(matrix, group)

        self.bits = bits
        self.head = quantize(self.embed)
        self.layers = []
        blocks, shared = -(-max_tokens // block_tokens), -(-shared_tokens // block_tokens)
        for w in weights["layers"]:
            self.layers.append(dict(
                in_norm=w["in_norm"], post_norm=w["post_norm"],
                qkv=quantize(torch.cat((w["q"], w["k"], w["v"]))),
                o=quantize(w["o"]),
                gate_up=quantize(torch.cat((w["gate"], w["up"]))),
                down=quantize(w["down"]),
                cache=serve.Kv8Cache(seqs * blocks + shared, block_tokens, kv_heads, head_dim, fmt, device=dev)))
        # sequence b owns blocks b, b + seqs, ...
        self.table = torch.arange(seqs * blocks, dtype=torch.int32, device=dev).view(blocks, seqs).t().contiguous()
        self.lengths = torch.zeros(seqs, dtype=torch.int32, device=dev)
        self.unknown = torch.zeros(seqs, 1, dtype=torch.bool, device=dev)   # sequences with ids outside the vocabulary
        # the prefix the blocks behind them
        self.shared_tokens, self.shared_blocks = shared_tokens, torch.arange(
            seqs * blocks, seqs * blocks + shared, dtype=torch.int32, device=dev)
        self.shared_length = torch.zeros(1, dtype=torch.int32, device=dev)
        self.shared_unknown = torch.zeros(1, 1, dtype=torch.bool, device=dev)
        inv = 1.0 / rope_theta ** (torch.arange(0, head_dim, 2, device=dev, dtype=torch.float32) / head_dim)
        angle = torch.outer(torch.arange(shared_tokens + max_tokens, device=dev, dtype=torch.float32), inv)
        self.cos, self.sin = angle.cos(), angle.sin()

    def _lookup(self, ids: torch.Tensor, mark: torch.Tensor | None = None) -> torch.Tensor:
        """Rows of the embedding for ids [seqs, n]: NaN for a sequence with an id outside the vocabulary, which ``mark``
        [seqs, 1] notes too, since not every layer kernel keeps a NaN."""
        held = ids.clamp(0, self.embed.shape[0] - 1)
        unknown = (held != ids).any(1, keepdim=True)
        if mark is not None:
            mark |= unknown
        return self.embed[held.flatten()].masked_fill_(unknown.expand_as(ids).reshape(-1, 1), float("nan"))

    def _norm(self, x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
        y, var = torch.empty_like(x), torch.empty(x.shape[0], device=x.device)
        check(lib.glt_rmsnorm_fwd(_p(x), _p(w), _p(y), _p(var), x.shape[0], x.shape[1], self.eps,
                                  torch.cuda.current_stream().cuda_stream))
        return y

    def _project(self, weight, x: torch.Tensor, norm: torch.Tensor, **kw) -> torch.Tensor:
        """The weight's product with the RMSNorm of x; 8-bit products take the norm with the quantisation."""
        if self.bits == 8:
            return weight.linear(x, norm=norm, eps=self.eps, **kw)
        return weight.linear(self._norm(x, norm), **kw)

    def _rope(self, qk: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
        """Half-split rotation of [rows, heads, head_dim] at the rows' own positions."""
        a, b = qk.float().chunk(2, -1)
        c, s = self.cos[pos][:, None], self.sin[pos][:, None]
        return torch.cat((a * c - b * s, a * s + b * c), -1).to(torch.bfloat16)

    def _swiglu(self, gate_up: torch.Tensor) -> torch.Tensor:
        rows, two = gate_up.shape
        half = two // 2
        h = torch.empty(rows, half, dtype=gate_up.dtype, device=gate_up.device)
        check(lib.glt_swiglu_fwd(_p(gate_up), C.c_void_p(gate_up.data_ptr() + 2 * half), _p(h), rows, half, two, two,
                                 half, torch.cuda.current_stream().cuda_stream))
        return h

    def share(self, ids: torch.Tensor) -> None:
        """Runs the prompt ids [n] that all sequences begin with, in place of an earlier one.  The sequences
        must be empty."""
        if ids.dim() != 1 or not 1 <= ids.shape[0] <= self.shared_tokens or ids.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"a shared prompt must be int32 or int64 [1 to shared_tokens {self.shared_tokens}], "
                             f"got {ids.dtype} {tuple(ids.shape)}")
        if self.held:
            raise ValueError(f"the sequences hold {self.held} tokens behind their prefix already")
        with torch.cuda.device(self.embed.device):
            self.prefix = None
            self.shared_length.zero_()
            self.shared_unknown.zero_()
            self._layers(ids[None], serve.Kv8Batch(self.shared_blocks[None], self.shared_length, ids.numel()),
                         torch.arange(ids.numel(), device=ids.device), self.shared_unknown)
            self.shared_length += ids.numel()
        self.prefix = serve.Kv8Prefix(self.shared_blocks, self.shared_length)

    def reset(self) -> None:
        """Starts over with empty sequences; a shared prefix stays."""
        self.lengths.zero_()
        if self.unknown is not None:
            self.unknown.zero_()
        self.held = 0

    def _fits(self, ids: torch.Tensor, more: int = 0) -> None:
        """Refuses what the cache and the rotary table have no room for: ids [seqs, n] and `more` tokens after them."""
        if ids.dim() != 2 or ids.shape[0] != self.seqs or ids.shape[1] < 1 or ids.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"ids must be int32 or int64 [{self.seqs}, at least 1], got {ids.dtype} {tuple(ids.shape)}")
        n = ids.shape[1] + more
        if self.held + n > self.max_tokens:
            raise ValueError(f"{n} tokens after the {self.held} held are more than max_tokens {self.max_tokens}")

    def step(self, ids: torch.Tensor) -> torch.Tensor:
        """New tokens ids [seqs, n] of every sequence: fp32 logits [seqs, vocab] after the last one."""
        self._fits(ids)
        with torch.cuda.device(self.embed.device):   # the layer kernels take the current one
            logits = self._step(ids)
        self.held += ids.shape[1]
        return logits

    def _step(self, ids: torch.Tensor) -> torch.Tensor:
        n = ids.shape[1]
        pos = self.lengths[:, None] + torch.arange(n, device=ids.device)
        if self.prefix is not None:
            pos = pos + self.shared_length
        x = self._layers(ids, serve.Kv8Batch(self.table, self.lengths, ids.numel()), pos.flatten(), self.unknown)
        self.lengths += n
        last = x.view(self.seqs, n, -1)[:, -1].contiguous()
        unknown = self.unknown if self.prefix is None else self.unknown | self.shared_unknown
        return self._project(self.head, last, self.final_norm, out_dtype=torch.float32).masked_fill_(unknown, float("nan"))

    def _layers(self, ids: torch.Tensor, batch: serve.Kv8Batch, pos: torch.Tensor, mark: torch.Tensor) -> torch.Tensor:
        """The layers' output [rows, hidden] of the batch's new tokens at positions pos [rows]; ``mark`` as for _lookup."""
        hd, x = self.head_dim, self._lookup(ids, mark)
        for w in self.layers:
            qkv = self._project(w["qkv"], x, w["in_norm"]).unflatten(1, (-1, hd))
            rotated = self._rope(qkv[:, :self.heads + self.kv_heads], pos)
            w["cache"].append(batch, rotated[:, self.heads:], qkv[:, self.heads + self.kv_heads:])
            if self.prefix is not None:
                o, _ = w["cache"].prefix_attention(batch, self.prefix, rotated[:, :self.heads])
            else:
                o, _ = w["cache"].attention(batch, rotated[:, :self.heads], window=self.window, sinks=self.sinks)
            x = w["o"].linear(o.flatten(1), resid=x)
            h = self._swiglu(self._project(w["gate_up"], x, w["post_norm"]))
            x = w["down"].linear(h, resid=x)
        return x

    def generate(self, prompt: torch.Tensor, tokens: int):
        """Greedy continuation of prompt [seqs, n]: (ids [seqs, tokens], log probabilities)."""
        if tokens < 1:
            raise ValueError(f"{tokens} tokens to generate (at least 1)")
        self._fits(prompt, tokens - 1)   # the last one is not fed back
        ids, logps = [], []
        logits = self.step(prompt)
        for i in range(tokens):
            r = serve.token_logprobs(logits, top=1)
            ids.append(r.top_ids)
            logps.append(r.top_logp)
            if i + 1 < tokens:
                logits = self.step(r.top_ids)
        return torch.cat(ids, 1), torch.cat(logps, 1)


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--seqs", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=256)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--bits", type=int, choices=(4, 8), default=4)
    ap.add_argument("--shared", type=int, default=0, help="tokens of a prompt that all sequences begin with")
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=0)
    a = ap.parse_args()
    if min(a.seqs, a.prompt, a.tokens) < 1:
        ap.error("--seqs, --prompt and --tokens must be at least 1")
    if min(a.shared, a.window, a.sinks) < 0 or (a.window and a.shared) or (a.sinks and not a.window):
        ap.error("--shared and --window exclude each other, and --sinks needs --window")
    w = random_weights(hidden=896, intermediate=4864, layers=24, heads=14, kv_heads=2, head_dim=64, vocab=151936)
    d = Decoder(w, heads=14, kv_heads=2, head_dim=64, seqs=a.seqs, max_tokens=a.prompt + a.tokens, bits=a.bits, shared_tokens=a.shared,
                window=a.window, sinks=a.sinks)
    if a.shared:
        d.share(torch.randint(0, 151936, (a.shared,), device="cuda", dtype=torch.int32))
    prompt = torch.randint(0, 151936, (a.seqs, a.prompt), device="cuda", dtype=torch.int32)
    d.generate(prompt, 2)   # first calls load their kernels
    d.reset()
    torch.cuda.synchronize()
    t = time.perf_counter()
    ids, logps = d.generate(prompt, a.tokens)
    torch.cuda.synchronize()
    t = time.perf_counter() - t
    code = C.c_uint()
    check(lib.glt_device_error(C.byref(code)))
    if code.value:
        raise RuntimeError(f"device error word {code.value}")
    print(f"{a.seqs} sequences, prompt {a.prompt}: {a.seqs * a.tokens / t:.0f} tokens/s "
          f"({1e3 * t / a.tokens:.2f} ms a step), mean log probability {logps.mean().item():.3f}")


if __name__ == "__main__":
    main()
