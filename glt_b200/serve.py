"""Decoding and scoring with a (baked) model, over the C ABI.

``Kv8Cache`` / ``Kv8Batch``: a key/value cache in 8 bits with one scale for each block of
tokens and head, and the attention that reads it; ``W4Weight``: products with 4-bit weights
and group scales; ``W8Weight`` / ``quantize_rows``: products in 8-bit integers with a scale for each
token and channel; ``token_logprobs`` / ``token_logprobs_bwd``: log probabilities of given
tokens, entropy, the most likely tokens, and the gradient.  Every call runs on the device that its
tensors share (which need not be the current one), on its current stream, allocates its outputs
with torch and does not synchronise.
``include/glt_graft.h`` states the formulas, ranges and errors.
"""
from __future__ import annotations

import ctypes as C
import threading
from typing import NamedTuple

import torch

from ._lib import GltKv8Batch as _CBatch, GltKv8Cache as _CCache, GltKv8Prefix as _CPrefix, check, lib

FORMATS = {"int8": 0, "e4m3": 1}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)   # the handle without a Stream object around it
_capturing = torch.cuda.is_current_stream_capturing
_current_device = torch.cuda.current_device
_BF16, _F32, _I32, _U8, _I8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8, torch.int8


def _stream(i: int) -> int:
    """The current stream of device i."""
    return _raw_stream(i) if _raw_stream is not None else torch.cuda.current_stream(i).cuda_stream


def _one_device(**tensors: torch.Tensor | None) -> int:
    """The CUDA device that all of them lie on."""
    at = {n: t.get_device() for n, t in tensors.items() if t is not None}
    i = next(iter(at.values()))
    if i < 0 or any(j != i for j in at.values()):
        raise ValueError(f"{', '.join(at)} must lie on one CUDA device")
    return i


class _Scratch(threading.local):
    """Workspaces of one host thread, one for each device and stream.  A call may be two launches that share its
    workspace: a thread's calls on a stream run in order and may share one too, but another thread's may come
    between the two.  A call under capture gets its own, since graphs may replay side by side."""

    def __init__(self):
        self._held: dict[tuple[int, int], torch.Tensor] = {}

    def get(self, nbytes: int, device: int, stream: int) -> torch.Tensor:
        ws = self._held.get((device, stream))
        if ws is None or ws.numel() < nbytes or _capturing():
            ws = torch.empty(max(nbytes, 16), dtype=_U8, device=torch.device("cuda", device))
            if not _capturing():
                self._held[device, stream] = ws
        return ws


_scratch = _Scratch()


def _need(ok: bool, msg: str) -> None:
    if not ok:
        raise ValueError(msg)


def _int32(t: torch.Tensor, name: str) -> torch.Tensor:
    if not (t.is_cuda and t.dtype is _I32 and t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous int32 CUDA tensor")
    return t


def _rows(t: torch.Tensor, device: int, rows: int, heads: int, hd: int, name: str) -> int:
    """Row stride of a bf16 [rows, heads, hd] tensor of the device whose rows are dense."""
    if not (t.get_device() == device and t.dtype is _BF16 and t.shape == (rows, heads, hd)):
        raise ValueError(f"{name} must be a bf16 tensor [{rows}, {heads}, {hd}] on cuda:{device}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    s = t.stride()
    if (s[2] != 1 or (s[1] != hd and heads > 1)) and t.numel():
        raise ValueError(f"{name}: a row's heads must be contiguous")
    return s[0] if rows > 1 else heads * hd


class Kv8Batch:
    """One step of a batch of sequences, shared by all layers (GltKv8Batch).

    block_table int32 [num_seqs, max_blocks]; lengths int32 [num_seqs], the tokens held
    before this step; rows, the step's new rows in all; row_start int32 [num_seqs + 1] when the
    sequences bring different numbers of rows; max_new, the most any of them brings."""

    def __init__(self, block_table: torch.Tensor, lengths: torch.Tensor, rows: int,
                 row_start: torch.Tensor | None = None, max_new: int | None = None):
        _need(block_table.dim() == 2 and lengths.shape == block_table.shape[:1],
              "block_table [num_seqs, max_blocks] and lengths [num_seqs]")
        n = block_table.shape[0]
        _need(row_start is None or row_start.shape == (n + 1,), "row_start [num_seqs + 1]")
        if max_new is None:
            max_new = rows if row_start is not None else rows // max(n, 1)
        self.block_table, self.lengths = _int32(block_table, "block_table"), _int32(lengths, "lengths")
        self.row_start = None if row_start is None else _int32(row_start, "row_start")
        self._device = _one_device(block_table=block_table, lengths=lengths, row_start=row_start)
        self.num_seqs, self.max_blocks, self.rows = n, block_table.shape[1], rows
        self._c = _CBatch(n, self.max_blocks, rows, max_new, block_table.data_ptr(), lengths.data_ptr(),
                          None if row_start is None else row_start.data_ptr())
        self._p = C.byref(self._c)
        self._ws_bytes: dict[tuple, int] = {}   # attention's workspace by what it depends on


class Kv8Prefix:
    """A prefix that all sequences of a batch share, for all layers (GltKv8Prefix).

    blocks int32 [n], the blocks of the cache that hold it; length int32 [1], its tokens (read on the device)."""

    def __init__(self, blocks: torch.Tensor, length: torch.Tensor):
        _need(blocks.dim() == 1 and length.shape == (1,), "blocks [n] and length [1]")
        self.blocks, self.length = _int32(blocks, "blocks"), _int32(length, "length")
        self._device = _one_device(blocks=blocks, length=length)
        self._c = _CPrefix(blocks.shape[0], blocks.data_ptr(), length.data_ptr())
        self._p = C.byref(self._c)


class Kv8Cache:
    """One layer's key/value cache in 8 bits (GltKv8Cache)."""

    def __init__(self, num_blocks: int, block_tokens: int, num_kv_heads: int, head_dim: int, fmt: str = "int8",
                 device="cuda"):
        shape = (num_blocks, num_kv_heads, block_tokens, head_dim)
        self._bind(torch.empty(shape, dtype=torch.uint8, device=device),
                   torch.empty(shape, dtype=torch.uint8, device=device),
                   torch.empty(shape[:2], device=device), torch.empty(shape[:2], device=device), fmt)

    @classmethod
    def from_buffers(cls, k, v, k_scale, v_scale, fmt: str = "int8") -> "Kv8Cache":
        """A cache over the caller's buffers: codes uint8 [num_blocks, num_kv_heads, block_tokens,
        head_dim], scales fp32 [num_blocks, num_kv_heads]."""
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale, fmt)
        return self

    def _bind(self, k, v, k_scale, v_scale, fmt):
        _need(fmt in FORMATS, f"format {fmt!r} (one of {sorted(FORMATS)})")
        _need(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype == torch.uint8,
              "codes must be uint8 [num_blocks, num_kv_heads, block_tokens, head_dim]")
        _need(k_scale.shape == v_scale.shape == k.shape[:2] and k_scale.dtype == v_scale.dtype == torch.float32,
              "scales must be fp32 [num_blocks, num_kv_heads]")
        _need(all(t.is_cuda and t.is_contiguous() for t in (k, v, k_scale, v_scale)),
              "cache buffers must be contiguous CUDA tensors")
        self._device = _one_device(k=k, v=v, k_scale=k_scale, v_scale=v_scale)
        self.k, self.v, self.k_scale, self.v_scale, self.fmt = k, v, k_scale, v_scale, fmt
        self.num_blocks, self.num_kv_heads, self.block_tokens, self.head_dim = k.shape
        self._c = _CCache(FORMATS[fmt], self.block_tokens, self.num_kv_heads, self.head_dim, self.num_blocks,
                          k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr())
        self._p = C.byref(self._c)

    def _batch_device(self, batch: Kv8Batch) -> int:
        if batch._device != self._device:
            raise ValueError(f"the cache lies on cuda:{self._device}, the batch on cuda:{batch._device}")
        return self._device

    def append(self, batch: Kv8Batch, k: torch.Tensor, v: torch.Tensor) -> None:
        """Write the step's keys and values, bf16 [rows, num_kv_heads, head_dim] (views into packed rows are fine)."""
        dev = self._batch_device(batch)
        if dev != _current_device():
            with torch.cuda.device(dev):
                return self.append(batch, k, v)
        ld_k = _rows(k, dev, batch.rows, self.num_kv_heads, self.head_dim, "k")
        ld_v = _rows(v, dev, batch.rows, self.num_kv_heads, self.head_dim, "v")
        st = lib.glt_kv8_append(self._p, batch._p, k.data_ptr(), ld_k, v.data_ptr(), ld_v, _stream(dev))
        if st:
            check(st)

    def _step(self, batch: Kv8Batch, q: torch.Tensor, token_mask: torch.Tensor | None, out: torch.Tensor | None):
        """Checks what every form of attention takes: (ld_q, out, ld_o, lse, mask's address, its row stride)."""
        dev, rows, nh = self._device, batch.rows, q.shape[1]
        ld_q = _rows(q, dev, rows, nh, self.head_dim, "q")
        if out is None:
            out = torch.empty(q.shape, dtype=_BF16, device=q.device)
            ld_o = nh * self.head_dim
        else:
            ld_o = _rows(out, dev, rows, nh, self.head_dim, "out")
        lse = torch.empty((rows, nh), dtype=_F32, device=q.device)
        mask, ld_m = None, 0
        if token_mask is not None:
            width = batch.max_blocks * self.block_tokens
            if not (token_mask.get_device() == dev and token_mask.dtype in (torch.uint8, torch.bool)
                    and token_mask.dim() == 2 and token_mask.shape[0] == batch.num_seqs and token_mask.stride(1) == 1
                    and token_mask.shape[1] >= width):
                raise ValueError(f"token_mask must be bytes [{batch.num_seqs}, at least {width}] on cuda:{dev}")
            mask = token_mask.data_ptr()
            ld_m = token_mask.stride(0) if token_mask.shape[0] > 1 else token_mask.shape[1]
        return ld_q, out, ld_o, lse, mask, ld_m

    def attention(self, batch: Kv8Batch, q: torch.Tensor, scale: float = 0.0, window: int = 0,
                  token_mask: torch.Tensor | None = None, out: torch.Tensor | None = None, sinks: int = 0):
        """Attention of the step's queries, bf16 [rows, num_heads, head_dim], after ``append``.  With a window, the
        first ``sinks`` tokens of a sequence stay visible behind it.
        Returns (o like q, dense; lse fp32 [rows, num_heads])."""
        if q.dim() != 3:
            raise ValueError("q must be [rows, num_heads, head_dim]")
        dev = self._batch_device(batch)
        if dev != _current_device():
            with torch.cuda.device(dev):
                return self.attention(batch, q, scale, window, token_mask, out, sinks)
        nh = q.shape[1]
        ld_q, out, ld_o, lse, mask, ld_m = self._step(batch, q, token_mask, out)
        key = (nh, self.num_kv_heads, self.block_tokens, self.head_dim)
        need = batch._ws_bytes.get(key)
        if need is None:
            n = C.c_int64()
            check(lib.glt_kv8_attention_workspace(self._p, batch._p, nh, C.byref(n)))
            need = batch._ws_bytes[key] = n.value
        stream = _stream(dev)
        ws = _scratch.get(need, dev, stream)
        if sinks:
            st = lib.glt_kv8_window_attention(self._p, batch._p, q.data_ptr(), ld_q, out.data_ptr(), ld_o, lse.data_ptr(),
                                              nh, scale, window, sinks, mask, ld_m, ws.data_ptr(), need, stream)
        else:
            st = lib.glt_kv8_attention(self._p, batch._p, q.data_ptr(), ld_q, out.data_ptr(), ld_o, lse.data_ptr(), nh,
                                       scale, window, mask, ld_m, ws.data_ptr(), need, stream)
        if st:
            check(st)
        return out, lse

    def prefix_attention(self, batch: Kv8Batch, prefix: Kv8Prefix, q: torch.Tensor, scale: float = 0.0,
                         token_mask: torch.Tensor | None = None, out: torch.Tensor | None = None):
        """``attention`` in which every sequence of the batch is the prefix followed by its own tokens, which alone the
        batch's tables and lengths (and ``token_mask``) describe."""
        if q.dim() != 3:
            raise ValueError("q must be [rows, num_heads, head_dim]")
        dev = self._batch_device(batch)
        if prefix._device != dev:
            raise ValueError(f"the cache lies on cuda:{dev}, the prefix on cuda:{prefix._device}")
        if dev != _current_device():
            with torch.cuda.device(dev):
                return self.prefix_attention(batch, prefix, q, scale, token_mask, out)
        nh = q.shape[1]
        ld_q, out, ld_o, lse, mask, ld_m = self._step(batch, q, token_mask, out)
        key = (nh, self.num_kv_heads, self.block_tokens, self.head_dim, prefix.blocks.shape[0])
        need = batch._ws_bytes.get(key)
        if need is None:
            n = C.c_int64()
            check(lib.glt_kv8_prefix_attention_workspace(self._p, batch._p, prefix._p, nh, C.byref(n)))
            need = batch._ws_bytes[key] = n.value
        stream = _stream(dev)
        ws = _scratch.get(need, dev, stream)
        st = lib.glt_kv8_prefix_attention(self._p, batch._p, prefix._p, q.data_ptr(), ld_q, out.data_ptr(), ld_o,
                                          lse.data_ptr(), nh, scale, mask, ld_m, ws.data_ptr(), need, stream)
        if st:
            check(st)
        return out, lse

    def read(self, batch: Kv8Batch, start: torch.Tensor | None, count: int):
        """Cached values of positions [start[b], start[b] + count): two fp32 tensors
        [num_seqs, count, num_kv_heads, head_dim]."""
        dev = self._batch_device(batch)
        if dev != _current_device():
            with torch.cuda.device(dev):
                return self.read(batch, start, count)
        if start is not None:
            _need(_int32(start, "start").shape == (batch.num_seqs,) and start.get_device() == dev,
                  f"start [num_seqs] on cuda:{dev}")
        shape = (batch.num_seqs, count, self.num_kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=_F32, device=self.k.device)
        v = torch.empty(shape, dtype=_F32, device=self.k.device)
        st = lib.glt_kv8_read(self._p, batch._p, None if start is None else start.data_ptr(), count, k.data_ptr(),
                              v.data_ptr(), _stream(dev))
        if st:
            check(st)
        return k, v


def _packed_bytes(N: int, K: int, group: int, asym: bool) -> int:
    n = C.c_int64()
    check(lib.glt_w4_packed_bytes(N, K, group, int(asym), C.byref(n)))
    return n.value


class W4Weight:
    """A weight matrix [N, K] in 4 bits with group scales, packed for ``linear``."""

    def __init__(self, packed: torch.Tensor, N: int, K: int, group: int, asym: bool):
        need = _packed_bytes(N, K, group, asym)
        _need(packed.is_cuda and packed.dtype is _U8 and packed.dim() == 1 and packed.is_contiguous()
              and packed.numel() >= need, f"packed must be a contiguous uint8 CUDA tensor of at least {need} bytes")
        self._device = packed.get_device()
        self.packed, self.N, self.K, self.group, self.asym = packed, N, K, group, bool(asym)
        self._ws_bytes: dict[tuple, int] = {}

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None) -> "W4Weight":
        """codes uint8 [N, K] (0..15), scales bf16 [N, K / group], zeros uint8 like the scales or None (8)."""
        dev = _one_device(codes=codes, scales=scales, zeros=zeros)
        if dev != _current_device():
            with torch.cuda.device(dev):
                return cls.from_codes(codes, scales, zeros)
        _need(codes.dim() == 2, "codes [N, K]")
        N, K = codes.shape
        _need(scales.dim() == 2 and scales.shape[0] == N and scales.shape[1] > 0 and K % scales.shape[1] == 0,
              "scales must be [N, K / group]")
        group = K // scales.shape[1]
        _need(codes.dtype == torch.uint8 and scales.dtype == torch.bfloat16, "codes uint8, scales bf16")
        _need(zeros is None or (zeros.dtype == torch.uint8 and zeros.shape == scales.shape), "zeros uint8 like scales")
        codes, scales = codes.contiguous(), scales.contiguous()
        zeros = None if zeros is None else zeros.contiguous()
        packed = torch.empty(_packed_bytes(N, K, group, zeros is not None), dtype=torch.uint8, device=codes.device)
        check(lib.glt_w4_pack(codes.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(), N, K,
                              group, packed.data_ptr(), _stream(dev)))
        return cls(packed, N, K, group, zeros is not None)

    @classmethod
    def quantize(cls, w: torch.Tensor, group: int = 128, asym: bool = False) -> "W4Weight":
        """Round a bf16 [N, K] matrix to 4 bits."""
        return cls.from_codes(*quantize_w4(w, group, asym))

    def unpack(self) -> torch.Tensor:
        """The weights the codes stand for, bf16 [N, K]."""
        dev = self._device
        if dev != _current_device():
            with torch.cuda.device(dev):
                return self.unpack()
        w = torch.empty(self.N, self.K, dtype=torch.bfloat16, device=self.packed.device)
        check(lib.glt_w4_unpack(self.packed.data_ptr(), self.N, self.K, self.group, int(self.asym), w.data_ptr(),
                                self.K, _stream(dev)))
        return w

    def linear(self, x: torch.Tensor, resid: torch.Tensor | None = None,
               out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
        """x . W^T (+ resid): x bf16 [M, K], result [M, N] in bf16 or fp32."""
        N, K, dev = self.N, self.K, self._device
        if dev != _current_device():
            with torch.cuda.device(dev):
                return self.linear(x, resid, out_dtype, out)
        if not (x.get_device() == dev and x.dtype is _BF16 and x.dim() == 2 and x.shape[1] == K and x.stride(1) == 1):
            raise ValueError(f"x must be a bf16 tensor [M, {K}] on cuda:{dev} with dense rows")
        M = x.shape[0]
        one = M <= 1
        if out is None:
            if out_dtype is not _BF16 and out_dtype is not _F32:
                raise ValueError("out_dtype must be bfloat16 or float32")
            out = torch.empty((M, N), dtype=out_dtype, device=x.device)
        elif not (out.get_device() == dev and out.shape == (M, N) and out.dtype in (_BF16, _F32) and out.stride(1) == 1):
            raise ValueError(f"out must be a bf16 or fp32 tensor [{M}, {N}] on cuda:{dev} with dense rows")
        bf16 = out.dtype is _BF16
        if resid is not None and not (resid.get_device() == dev and resid.dtype is _BF16 and resid.shape == (M, N) and
                                      resid.stride(1) == 1):
            raise ValueError(f"resid must be a bf16 tensor [{M}, {N}] on cuda:{dev} with dense rows")
        need = self._ws_bytes.get((M, bf16))
        if need is None:
            n = C.c_int64()
            check(lib.glt_w4_linear_workspace(M, N, K, self.group, bf16, C.byref(n)))
            need = self._ws_bytes[M, bf16] = n.value
        stream = _stream(dev)
        ws = _scratch.get(need, dev, stream)
        st = lib.glt_w4_linear(self.packed.data_ptr(), N, K, self.group, self.asym, x.data_ptr(),
                               K if one else x.stride(0), M, out.data_ptr(), N if one else out.stride(0), bf16,
                               None if resid is None else resid.data_ptr(),
                               0 if resid is None else N if one else resid.stride(0), ws.data_ptr(), need, stream)
        if st:
            check(st)
        return out


def quantize_w4(w: torch.Tensor, group: int = 128, asym: bool = False):
    """(codes uint8 [N, K], scales bf16 [N, K / group], zeros uint8 or None) of a bf16 matrix."""
    _need(w.is_cuda and w.dtype == torch.bfloat16 and w.dim() == 2 and w.stride(1) == 1, "w must be a bf16 CUDA matrix")
    dev = w.get_device()
    if dev != _current_device():
        with torch.cuda.device(dev):
            return quantize_w4(w, group, asym)
    N, K = w.shape
    _packed_bytes(N, K, group, asym)   # refuses sizes and groups that do not fit
    codes = torch.empty(N, K, dtype=torch.uint8, device=w.device)
    scales = torch.empty(N, K // group, dtype=torch.bfloat16, device=w.device)
    zeros = torch.empty(N, K // group, dtype=torch.uint8, device=w.device) if asym else None
    check(lib.glt_w4_quantize(w.data_ptr(), w.stride(0) if N > 1 else K, N, K, group, int(asym), codes.data_ptr(),
                              scales.data_ptr(), None if zeros is None else zeros.data_ptr(), _stream(dev)))
    return codes, scales, zeros


class W8Rows(NamedTuple):
    """Rows in 8 bits: codes int8 [rows, K], a view whose rows lie a multiple of 16 bytes apart with zeros between
    them, and scales fp32 [rows]."""
    codes: torch.Tensor
    scales: torch.Tensor


def _bf16_rows(t: torch.Tensor, device: int, rows: int | None, K: int, name: str) -> int:
    """Row stride of a bf16 [rows, K] tensor of the device whose rows are dense."""
    if not (t.get_device() == device and t.dtype is _BF16 and t.dim() == 2 and t.shape[1] == K and
            (rows is None or t.shape[0] == rows) and (t.stride(1) == 1 or K == 1)):
        raise ValueError(f"{name} must be a bf16 tensor [{'M' if rows is None else rows}, {K}] on cuda:{device} with dense rows")
    return t.stride(0) if t.shape[0] > 1 else K


def _norm_weight(norm: torch.Tensor | None, device: int, K: int) -> int | None:
    if norm is None:
        return None
    if not (norm.get_device() == device and norm.dtype is _BF16 and norm.shape == (K,) and norm.is_contiguous()):
        raise ValueError(f"norm must be a contiguous bf16 tensor [{K}] on cuda:{device}")
    return norm.data_ptr()


def quantize_rows(x: torch.Tensor, norm: torch.Tensor | None = None, eps: float = 1e-6) -> W8Rows:
    """Rows of bf16 x [rows, K] in 8 bits, each with its own scale; with ``norm`` (bf16 [K]) of its RMSNorm."""
    _need(x.is_cuda and x.dim() == 2 and x.shape[1] > 0, "x must be a bf16 CUDA tensor [rows, K]")
    dev = x.get_device()
    if dev != _current_device():
        with torch.cuda.device(dev):
            return quantize_rows(x, norm, eps)
    rows, K = x.shape
    ld_x, norm_at = _bf16_rows(x, dev, rows, K, "x"), _norm_weight(norm, dev, K)
    codes = torch.empty((rows, (K + 127) // 128 * 128), dtype=_I8, device=x.device)   # rows that begin with a line
    scales = torch.empty((rows,), dtype=_F32, device=x.device)
    check(lib.glt_w8_quantize_rows(x.data_ptr(), ld_x, rows, K, norm_at, eps, codes.data_ptr(), codes.shape[1],
                                   scales.data_ptr(), _stream(dev)))
    return W8Rows(codes[:, :K], scales)


class W8Weight:
    """A weight matrix [N, K] in 8-bit integers with a scale for each output channel."""

    def __init__(self, rows: W8Rows):
        codes, scales = rows
        _need(codes.is_cuda and codes.dtype is _I8 and codes.dim() == 2 and codes.shape[0] > 0 and codes.shape[1] > 0,
              "codes must be an int8 CUDA tensor [N, K]")
        self.N, self.K = codes.shape
        self._device = codes.get_device()
        _need(scales.get_device() == self._device and scales.dtype is _F32 and scales.shape == (self.N,)
              and scales.is_contiguous(), f"scales must be a contiguous fp32 tensor [{self.N}] on the codes' device")
        self._ld = codes.stride(0) if self.N > 1 else (self.K + 15) // 16 * 16
        if (codes.stride(1) != 1 and self.K > 1) or self._ld % 16 or self._ld < (self.K + 15) // 16 * 16:
            raise ValueError("rows of codes must be dense and lie a multiple of 16 bytes apart (from_codes lays any out)")
        self.codes, self.scales = codes, scales
        self._ws_bytes: dict[int, int] = {}

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor) -> "W8Weight":
        """codes int8 [N, K], scales fp32 [N]: the weight is codes * scales[:, None].  The codes are laid out anew."""
        _need(codes.is_cuda and codes.dtype is _I8 and codes.dim() == 2, "codes must be an int8 CUDA tensor [N, K]")
        _one_device(codes=codes, scales=scales)
        _need(scales.dtype is _F32, "scales must be fp32")
        N, K = codes.shape
        laid = torch.empty((N, (K + 127) // 128 * 128), dtype=_I8, device=codes.device)   # rows that begin with a line
        laid[:, :K] = codes
        laid[:, K:] = 0
        return cls(W8Rows(laid[:, :K], scales.contiguous()))

    @classmethod
    def quantize(cls, w: torch.Tensor) -> "W8Weight":
        """Round a bf16 [N, K] matrix to 8 bits, a scale for each row."""
        return cls(quantize_rows(w))

    def linear(self, x: torch.Tensor, resid: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16,
               out: torch.Tensor | None = None, norm: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
        """x . W^T (+ resid), x bf16 [M, K] rounded to 8 bits a row (after its RMSNorm with weight ``norm``);
        result [M, N] in bf16 or fp32."""
        K, dev = self.K, self._device
        if dev != _current_device():
            with torch.cuda.device(dev):
                return self.linear(x, resid, out_dtype, out, norm, eps)
        ld_x, norm_at = _bf16_rows(x, dev, None, K, "x"), _norm_weight(norm, dev, K)
        M = x.shape[0]
        out, ld_y, r, ld_r = self._outputs(M, resid, out_dtype, out)
        need = self._ws_bytes.get(M)
        if need is None:
            n = C.c_int64()
            check(lib.glt_w8_linear_workspace(M, K, C.byref(n)))
            need = self._ws_bytes[M] = n.value
        stream = _stream(dev)
        ws = _scratch.get(need, dev, stream)
        st = lib.glt_w8_linear(x.data_ptr(), ld_x, M, norm_at, eps, self.codes.data_ptr(), self._ld, self.scales.data_ptr(),
                               self.N, K, out.data_ptr(), ld_y, out.dtype is _BF16, r, ld_r, ws.data_ptr(), need, stream)
        if st:
            check(st)
        return out

    def linear_rows(self, rows: W8Rows, resid: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16,
                    out: torch.Tensor | None = None) -> torch.Tensor:
        """``linear`` of rows that ``quantize_rows`` gave, for weights that share their input."""
        K, dev = self.K, self._device
        if dev != _current_device():
            with torch.cuda.device(dev):
                return self.linear_rows(rows, resid, out_dtype, out)
        codes, scales = rows
        M = codes.shape[0]
        ld = codes.stride(0) if M > 1 else (K + 15) // 16 * 16
        if not (codes.get_device() == dev == scales.get_device() and codes.dtype is _I8 and codes.shape == (M, K) and
                (codes.stride(1) == 1 or K == 1) and scales.dtype is _F32 and scales.shape == (M,) and scales.is_contiguous()):
            raise ValueError(f"rows must be those quantize_rows gives of [M, {K}] on cuda:{dev}")
        out, ld_y, r, ld_r = self._outputs(M, resid, out_dtype, out)
        check(lib.glt_w8_linear_rows(codes.data_ptr(), ld, scales.data_ptr(), M, self.codes.data_ptr(), self._ld,
                                     self.scales.data_ptr(), self.N, K, out.data_ptr(), ld_y, out.dtype is _BF16, r, ld_r,
                                     _stream(dev)))
        return out

    def _outputs(self, M: int, resid, out_dtype, out):
        """(out, its row stride, resid's address, its row stride)"""
        N, dev = self.N, self._device
        if out is None:
            if out_dtype is not _BF16 and out_dtype is not _F32:
                raise ValueError("out_dtype must be bfloat16 or float32")
            out = torch.empty((M, N), dtype=out_dtype, device=self.codes.device)
        elif not (out.get_device() == dev and out.shape == (M, N) and out.dtype in (_BF16, _F32) and
                  (out.stride(1) == 1 or N == 1)):
            raise ValueError(f"out must be a bf16 or fp32 tensor [{M}, {N}] on cuda:{dev} with dense rows")
        r = ld_r = 0
        if resid is not None:
            ld_r, r = _bf16_rows(resid, dev, M, N, "resid"), resid.data_ptr()
        return out, out.stride(0) if M > 1 else N, r or None, ld_r


class TokenLogprobs(NamedTuple):
    logp: torch.Tensor | None      # fp32 [rows], None without targets
    entropy: torch.Tensor          # fp32 [rows]
    lse: torch.Tensor              # fp32 [rows]
    top_ids: torch.Tensor | None   # int32 [rows, top], None with top = 0
    top_logp: torch.Tensor | None  # fp32 [rows, top]
    scale: float


def _logits(x: torch.Tensor, device: int, name: str = "logits") -> tuple[bool, int]:
    """(whether bf16, row stride) of a [rows, V] tensor of the device."""
    if not (x.get_device() == device >= 0 and x.dim() == 2 and (x.dtype is _BF16 or x.dtype is _F32) and
            (x.stride(1) == 1 or x.shape[1] == 1)):
        raise ValueError(f"{name} must be a bf16 or fp32 CUDA tensor [rows, V] with dense rows, "
                         "all tensors of a call on one device")
    return x.dtype is _BF16, x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _per_row(t: torch.Tensor | None, device: int, rows: int, dtype: torch.dtype, name: str) -> int | None:
    """Address of a contiguous [rows] tensor of the device, None for None."""
    if t is None:
        return None
    if not (t.get_device() == device and t.dtype is dtype and t.shape == (rows,) and t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor [{rows}] on cuda:{device}")
    return t.data_ptr()


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor | None = None, scale: float = 1.0,
                   top: int = 0) -> TokenLogprobs:
    """Log probabilities of ``targets`` (int32 [rows], negative: none) under softmax(scale * logits),
    the entropy, and the ``top`` most likely tokens."""
    dev = logits.get_device()
    dt, ld = _logits(logits, dev)
    if dev != _current_device():
        with torch.cuda.device(dev):
            return token_logprobs(logits, targets, scale, top)
    R, V = logits.shape
    t = _per_row(targets, dev, R, _I32, "targets")
    stats = torch.empty((3, R), dtype=_F32, device=logits.device)
    at = stats.data_ptr()
    ids = vals = ids_at = vals_at = None
    if top > 0:
        ids = torch.empty((R, top), dtype=_I32, device=logits.device)
        vals = torch.empty((R, top), dtype=_F32, device=logits.device)
        ids_at, vals_at = ids.data_ptr(), vals.data_ptr()
    st = lib.glt_token_logprobs(logits.data_ptr(), dt, ld, R, V, t, scale, top, None if t is None else at, at + 4 * R,
                                at + 8 * R, ids_at, vals_at, _stream(dev))
    if st:
        check(st)
    logp, entropy, lse = stats.unbind()
    return TokenLogprobs(None if targets is None else logp, entropy, lse, ids, vals, scale)


def token_logprobs_bwd(logits: torch.Tensor, targets: torch.Tensor | None, fwd: TokenLogprobs,
                       d_logp: torch.Tensor | None = None, d_entropy: torch.Tensor | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of the logits from those of ``fwd.logp`` and ``fwd.entropy`` (fp32 [rows], None = 0);
    ``out`` may be the logits themselves."""
    dev = logits.get_device()
    dt, ld = _logits(logits, dev)
    if dev != _current_device():
        with torch.cuda.device(dev):
            return token_logprobs_bwd(logits, targets, fwd, d_logp, d_entropy, out)
    R, V = logits.shape
    if out is None:
        out = torch.empty((R, V), dtype=logits.dtype, device=logits.device)
        ld_o = V
    else:
        if out.shape != logits.shape or out.dtype is not logits.dtype:
            raise ValueError("out must have the logits' shape and dtype")
        ld_o = _logits(out, dev, "out")[1]
    st = lib.glt_token_logprobs_bwd(logits.data_ptr(), dt, ld, R, V, _per_row(targets, dev, R, _I32, "targets"), fwd.scale,
                                    _per_row(fwd.lse, dev, R, _F32, "fwd.lse"), _per_row(fwd.entropy, dev, R, _F32, "fwd.entropy"),
                                    _per_row(d_logp, dev, R, _F32, "d_logp"), _per_row(d_entropy, dev, R, _F32, "d_entropy"),
                                    out.data_ptr(), ld_o, _stream(dev))
    if st:
        check(st)
    return out
