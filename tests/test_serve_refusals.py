"""Arguments that the decoding and scoring calls refuse, on the host before any
launch (CPU only: the pointers are never followed)."""
import ctypes as C

import pytest

from glt_b200 import _lib
from glt_b200._lib import GltKv8Batch, GltKv8Cache, lib

EINVAL, OK = 1, 0
P = 1 << 20   # a 16-byte aligned address that nothing reads


def cache(**kw):
    d = dict(format=0, block_tokens=16, num_kv_heads=2, head_dim=64, num_blocks=8, k=P, v=P, k_scale=P, v_scale=P)
    d.update(kw)
    return C.byref(GltKv8Cache(**d))


def batch(**kw):
    d = dict(num_seqs=2, max_blocks=4, rows=2, max_new=1, block_table=P, lengths=P, row_start=None)
    d.update(kw)
    return C.byref(GltKv8Batch(**d))


def refused(status, *words):
    assert status == EINVAL
    for w in words:
        assert w in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(format=2), "format"), (dict(block_tokens=48), "block_tokens"), (dict(head_dim=96), "head_dim"),
    (dict(num_kv_heads=0), "num_kv_heads"), (dict(num_blocks=0), "num_blocks"), (dict(k=None), "null cache"),
    (dict(v=P + 8), "aligned"), (dict(v_scale=None), "null cache")])
def test_caches(kw, word):
    refused(lib.glt_kv8_append(cache(**kw), batch(), P, 128, P, 128, None), word)
    refused(lib.glt_kv8_attention(cache(**kw), batch(), P, 256, P, 256, None, 4, 0.0, 0, None, 0, None, 0, None), word)
    refused(lib.glt_kv8_read(cache(**kw), batch(), None, 1, P, P, None), word)


@pytest.mark.parametrize("kw,word", [
    (dict(num_seqs=-1), "num_seqs"), (dict(num_seqs=70000), "num_seqs"), (dict(rows=-2), "rows"),
    (dict(max_blocks=0), "max_blocks"), (dict(max_blocks=1 << 30), "max_blocks"), (dict(block_table=None), "null block table"),
    (dict(lengths=None), "lengths"), (dict(rows=3, max_new=2), "row_start"), (dict(rows=4), "max_new"),
    (dict(num_seqs=0), "without sequences"), (dict(max_new=-1), "max_new")])
def test_batches(kw, word):
    refused(lib.glt_kv8_append(cache(), batch(**kw), P, 128, P, 128, None), word)


def test_append_rows():
    for k, ld_k, v, ld_v in ((P, 120, P, 128), (P, 128, P, 132), (P + 2, 128, P, 128), (P, 128, P, 64)):
        refused(lib.glt_kv8_append(cache(), batch(), k, ld_k, v, ld_v, None), "aligned")
    refused(lib.glt_kv8_append(cache(), batch(), None, 128, P, 128, None), "null")
    assert lib.glt_kv8_append(cache(), batch(rows=0, max_new=0), None, 0, None, 0, None) == OK


def attend(c=None, b=None, q=P, ld_q=256, o=P, ld_o=256, nh=4, scale=0.0, window=0, mask=None, ld_m=0, ws=P, n=1 << 40):
    return lib.glt_kv8_attention(c or cache(), b or batch(), q, ld_q, o, ld_o, None, nh, scale, window, mask, ld_m, ws, n, None)


def test_attention():
    refused(attend(nh=3), "num_heads")
    refused(attend(nh=0), "num_heads")
    refused(attend(q=None), "null")
    refused(attend(ld_q=248), "aligned")
    refused(attend(o=P + 4), "aligned")
    refused(attend(scale=-1.0), "scale")
    refused(attend(scale=float("nan")), "scale")
    refused(attend(scale=float("inf")), "scale")
    refused(attend(window=-1), "window")
    refused(attend(mask=P, ld_m=63), "mask")
    assert attend(b=batch(rows=0, max_new=0), q=None, o=None) == OK
    need = C.c_int64()
    assert lib.glt_kv8_attention_workspace(cache(), batch(), 4, C.byref(need)) == OK and need.value >= 0
    if need.value:
        refused(attend(n=need.value - 1), "workspace")
        refused(attend(ws=P + 8), "workspace")
        refused(attend(ws=None), "workspace")
    refused(lib.glt_kv8_attention_workspace(cache(), batch(), 5, C.byref(need)), "num_heads")
    refused(lib.glt_kv8_attention_workspace(cache(), batch(), 4, None), "null")


def test_read():
    refused(lib.glt_kv8_read(cache(), batch(), None, -1, P, P, None), "count")
    refused(lib.glt_kv8_read(cache(), batch(), None, 1, None, P, None), "null")
    refused(lib.glt_kv8_read(cache(), batch(), None, 1, P, P + 4, None), "aligned")
    assert lib.glt_kv8_read(cache(), batch(), None, 0, None, None, None) == OK


@pytest.mark.parametrize("N,K,group", [(0, 64, 32), (4, 0, 32), (4, 96, 64), (4, 128, 16), (4, 256, 256)])
def test_w4_shapes(N, K, group):
    need = C.c_int64()
    refused(lib.glt_w4_packed_bytes(N, K, group, 0, C.byref(need)), "w4")
    refused(lib.glt_w4_quantize(P, max(K, 1), N, K, group, 0, P, P, None, None), "w4")
    refused(lib.glt_w4_pack(P, P, None, N, K, group, P, None), "w4")
    refused(lib.glt_w4_unpack(P, N, K, group, 0, P, max(K, 1), None), "w4")
    refused(lib.glt_w4_linear(P, N, K, group, 0, P, max(K, 8), 1, P, 64, 1, None, 0, P, 1 << 40, None), "w4")
    refused(lib.glt_w4_linear_workspace(1, N, K, group, 1, C.byref(need)), "w4")


def linear(x=P, ld_x=128, M=2, y=P, ld_y=40, yt=1, r=None, ld_r=0, packed=P, ws=P, n=1 << 40):
    return lib.glt_w4_linear(packed, 40, 128, 32, 0, x, ld_x, M, y, ld_y, yt, r, ld_r, ws, n, None)


def test_w4_arguments():
    refused(linear(x=None), "null")
    refused(linear(x=P + 2), "aligned")
    refused(linear(ld_x=132), "aligned")
    refused(linear(ld_x=120), "aligned")
    refused(linear(M=-1), "rows")
    refused(linear(yt=2), "type")
    refused(linear(ld_y=39), "stride")
    refused(linear(r=P, ld_r=39), "stride")
    refused(linear(packed=P + 8), "aligned")
    need = C.c_int64()
    assert lib.glt_w4_linear_workspace(2, 40, 128, 32, 1, C.byref(need)) == OK and need.value > 0
    refused(linear(n=need.value - 1), "workspace")
    refused(linear(ws=None), "workspace")
    refused(linear(ws=P + 8), "workspace")
    refused(lib.glt_w4_linear_workspace(-1, 40, 128, 32, 1, C.byref(need)), "rows")
    refused(lib.glt_w4_linear_workspace(2, 40, 128, 32, 1, None), "null")
    assert linear(M=0) == OK and linear(M=0, x=None, y=None, ws=None, n=0) == OK
    refused(lib.glt_w4_quantize(P, 128, 4, 128, 32, 1, P, P, None, None), "null")
    refused(lib.glt_w4_quantize(P, 127, 4, 128, 32, 0, P, P, None, None), "stride")
    refused(lib.glt_w4_packed_bytes(4, 128, 32, 0, None), "null")


def forward(x=P, dt=1, ld=100, R=2, V=100, t=P, scale=1.0, top=0, logp=P, lse=P, ids=None, vals=None):
    return lib.glt_token_logprobs(x, dt, ld, R, V, t, scale, top, logp, None, lse, ids, vals, None)


def backward(x=P, dt=1, ld=100, R=2, V=100, t=P, scale=1.0, lse=P, ent=P, dl=P, de=None, d=P + (1 << 19), ld_d=100):
    return lib.glt_token_logprobs_bwd(x, dt, ld, R, V, t, scale, lse, ent, dl, de, d, ld_d, None)


def test_token_logprobs():
    refused(forward(x=None), "null")
    refused(forward(lse=None), "null")
    refused(forward(dt=2), "dtype")
    refused(forward(R=-1), "rows")
    refused(forward(V=0), "V 0")
    refused(forward(ld=99), "ld")
    refused(forward(x=P + 1), "aligned")
    refused(forward(dt=0, x=P + 2), "aligned")
    for s in (0.0, -1.0, float("nan"), float("inf")):
        refused(forward(scale=s), "scale")
        refused(backward(scale=s), "scale")
    refused(forward(top=33, V=100, ids=P, vals=P), "top")
    refused(forward(top=5, V=4, ld=4, ids=P, vals=P), "top")
    refused(forward(top=-1), "top")
    refused(forward(top=3), "top")
    refused(forward(logp=None), "targets")
    refused(forward(t=None), "targets")
    assert forward(R=0) == OK and forward(R=0, x=None, lse=None, top=3) == OK


def test_token_logprobs_backward():
    refused(backward(d=None), "null")
    refused(backward(lse=None), "null")
    refused(backward(dt=3), "dtype")
    refused(backward(ld_d=99), "ld_d")
    refused(backward(t=None), "targets")
    refused(backward(ent=None, de=P), "entropy")
    refused(backward(d=P + 1), "aligned")
    refused(backward(d=P, ld_d=104), "in place")
    assert backward(R=0) == OK
