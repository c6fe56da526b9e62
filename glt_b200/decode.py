"""Greedy decoding of a decoder whose projections are in 4 bits and whose key/value cache is in 8,
built from the operators of ``glt_b200.serve`` and the layer kernels of the C ABI.

``Decoder`` takes the (baked) bf16 weights of a model, rounds its projections to 4 bits and keeps a
cache for a batch of sequences; ``step`` runs any number of new tokens of each sequence (a
prompt or one token) and returns the logits of the last one; ``generate`` decodes and returns
the tokens with their log probabilities.

Usage:  python -m glt_b200.decode [--seqs N] [--prompt N] [--tokens N]
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
    """A decoder over 4-bit projections (the head is the embedding's transpose) and an 8-bit cache.

    The cache holds ``seqs`` sequences of up to ``max_tokens`` tokens; ``lengths`` counts the tokens
    each one has on the device, ``held`` on the host.  ``reset`` forgets them."""

    def __init__(self, weights: dict, heads: int, kv_heads: int, head_dim: int, seqs: int, max_tokens: int,
                 group: int = 64, block_tokens: int = 64, fmt: str = "int8", rope_theta: float = 1e6,
                 eps: float = 1e-6):
        self.heads, self.kv_heads, self.head_dim, self.seqs, self.eps = heads, kv_heads, head_dim, seqs, eps
        self.max_tokens, self.held = max_tokens, 0
        self.embed, self.final_norm = weights["embed"], weights["final_norm"]
        dev = self.embed.device
        self.head = serve.W4Weight.quantize(self.embed, group)
        self.layers = []
        blocks = -(-max_tokens // block_tokens)
        for w in weights["layers"]:
            self.layers.append(dict(
                in_norm=w["in_norm"], post_norm=w["post_norm"],
                qkv=serve.W4Weight.quantize(torch.cat((w["q"], w["k"], w["v"])), group),
                o=serve.W4Weight.quantize(w["o"], group),
                gate_up=serve.W4Weight.quantize(torch.cat((w["gate"], w["up"])), group),
                down=serve.W4Weight.quantize(w["down"], group),
                cache=serve.Kv8Cache(seqs * blocks, block_tokens, kv_heads, head_dim, fmt, device=dev)))
        # sequence b owns blocks b, b + seqs, ...
        self.table = torch.arange(seqs * blocks, dtype=torch.int32, device=dev).view(blocks, seqs).t().contiguous()
        self.lengths = torch.zeros(seqs, dtype=torch.int32, device=dev)
        inv = 1.0 / rope_theta ** (torch.arange(0, head_dim, 2, device=dev, dtype=torch.float32) / head_dim)
        angle = torch.outer(torch.arange(max_tokens, device=dev, dtype=torch.float32), inv)
        self.cos, self.sin = angle.cos(), angle.sin()

    def _lookup(self, ids: torch.Tensor) -> torch.Tensor:
        """Rows of the embedding for ids [seqs, n].  A sequence with an id outside the vocabulary gets NaN, which
        its logits and log probabilities show: the host does not wait to look at the ids."""
        held = ids.clamp(0, self.embed.shape[0] - 1)
        unknown = (held != ids).any(1, keepdim=True).expand_as(ids).reshape(-1, 1)
        return self.embed[held.flatten()].masked_fill_(unknown, float("nan"))

    def _norm(self, x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
        y, var = torch.empty_like(x), torch.empty(x.shape[0], device=x.device)
        check(lib.glt_rmsnorm_fwd(_p(x), _p(w), _p(y), _p(var), x.shape[0], x.shape[1], self.eps,
                                  torch.cuda.current_stream().cuda_stream))
        return y

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

    def reset(self) -> None:
        """Starts over with empty sequences."""
        self.lengths.zero_()
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
        n, hd = ids.shape[1], self.head_dim
        batch = serve.Kv8Batch(self.table, self.lengths, ids.numel())
        pos = (self.lengths[:, None] + torch.arange(n, device=ids.device)).flatten()
        x = self._lookup(ids)
        for w in self.layers:
            qkv = w["qkv"].linear(self._norm(x, w["in_norm"])).unflatten(1, (-1, hd))
            rotated = self._rope(qkv[:, :self.heads + self.kv_heads], pos)
            w["cache"].append(batch, rotated[:, self.heads:], qkv[:, self.heads + self.kv_heads:])
            o, _ = w["cache"].attention(batch, rotated[:, :self.heads])
            x = w["o"].linear(o.flatten(1), resid=x)
            h = self._swiglu(w["gate_up"].linear(self._norm(x, w["post_norm"])))
            x = w["down"].linear(h, resid=x)
        self.lengths += n
        last = x.view(self.seqs, n, -1)[:, -1].contiguous()
        return self.head.linear(self._norm(last, self.final_norm), out_dtype=torch.float32)

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
    a = ap.parse_args()
    if min(a.seqs, a.prompt, a.tokens) < 1:
        ap.error("--seqs, --prompt and --tokens must be at least 1")
    w = random_weights(hidden=896, intermediate=4864, layers=24, heads=14, kv_heads=2, head_dim=64, vocab=151936)
    d = Decoder(w, heads=14, kv_heads=2, head_dim=64, seqs=a.seqs, max_tokens=a.prompt + a.tokens)
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
