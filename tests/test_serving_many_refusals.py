"""What the 8-bit products, attention behind a prefix and windows with first tokens refuse, on the host before any launch
(CPU only: the pointers are never followed)."""
import ctypes as C
import sys
import threading

import pytest
import torch

from glt_b200 import _lib, decode, serve
from glt_b200._lib import GltKv8Batch, GltKv8Cache, GltKv8Prefix, lib
from serve_host import Host, on

EINVAL, OK = 1, 0
P = 1 << 20   # a 32-byte aligned address that nothing reads
BIG = 1 << 40


def cache(**kw):
    d = dict(format=0, block_tokens=16, num_kv_heads=2, head_dim=64, num_blocks=8, k=P, v=P, k_scale=P, v_scale=P)
    return C.byref(GltKv8Cache(**{**d, **kw}))


def batch(**kw):
    d = dict(num_seqs=2, max_blocks=4, rows=2, max_new=1, block_table=P, lengths=P, row_start=None)
    return C.byref(GltKv8Batch(**{**d, **kw}))


def prefix(**kw):
    return C.byref(GltKv8Prefix(**{**dict(num_blocks=3, block_ids=P, length=P), **kw}))


def refused(status, *words):
    assert status == EINVAL
    for w in words:
        assert w in _lib.last_error(), _lib.last_error()


def behind(c=None, b=None, p=None, q=P, ld_q=256, o=P, ld_o=256, nh=4, scale=0.0, mask=None, ld_m=0, ws=P, n=BIG):
    return lib.glt_kv8_prefix_attention(c or cache(), b or batch(), p or prefix(), q, ld_q, o, ld_o, None, nh, scale, mask, ld_m, ws, n, None)


def windowed(c=None, b=None, q=P, ld_q=256, o=P, ld_o=256, nh=4, scale=0.0, window=9, sinks=2, mask=None, ld_m=0, ws=P, n=BIG):
    return lib.glt_kv8_window_attention(c or cache(), b or batch(), q, ld_q, o, ld_o, None, nh, scale, window, sinks, mask, ld_m, ws, n, None)


@pytest.mark.parametrize("call", [behind, windowed])
def test_attention(call):
    refused(call(c=cache(format=2)), "format")
    refused(call(b=batch(lengths=None)), "lengths")
    refused(call(nh=3), "num_heads")
    refused(call(q=None), "null")
    refused(call(ld_q=248), "aligned")
    refused(call(o=P + 4), "aligned")
    for s in (-1.0, float("nan"), float("inf")):
        refused(call(scale=s), "scale")
    refused(call(mask=P, ld_m=63), "mask")
    refused(call(ws=None), "workspace")
    refused(call(ws=P + 8), "workspace")
    refused(call(n=15), "workspace")
    assert call(b=batch(rows=0, max_new=0), q=None, o=None) == OK


def test_windows():
    refused(windowed(window=-1), "window")
    refused(windowed(sinks=-1), "sinks")
    refused(windowed(sinks=0, window=-1), "window")


def test_prefixes():
    refused(behind(p=prefix(num_blocks=-1)), "prefix")
    refused(behind(p=prefix(num_blocks=1 << 30)), "prefix")
    refused(behind(p=prefix(block_ids=None)), "null prefix")
    refused(behind(p=prefix(length=None)), "null prefix")
    need = C.c_int64()
    refused(lib.glt_kv8_prefix_attention_workspace(cache(), batch(), None, 4, C.byref(need)), "null")
    refused(lib.glt_kv8_prefix_attention_workspace(cache(), batch(), prefix(), 4, None), "null")
    refused(lib.glt_kv8_prefix_attention_workspace(cache(), batch(), prefix(), 5, C.byref(need)), "num_heads")
    assert lib.glt_kv8_prefix_attention_workspace(cache(), batch(), prefix(), 4, C.byref(need)) == OK and need.value > 0
    refused(behind(n=need.value - 1), "workspace")
    refused(behind(ws=P + 16), "32-byte")
    own = C.c_int64()
    assert lib.glt_kv8_attention_workspace(cache(), batch(), 4, C.byref(own)) == OK and need.value > own.value
    refused(behind(b=batch(rows=1 << 28, max_new=1 << 28, num_seqs=1), nh=64, ld_q=1 << 13, ld_o=1 << 13), "rows")


def rows(x=P, ld=100, n=2, K=100, norm=None, eps=1e-6, codes=P, ld_c=112, scales=P):
    return lib.glt_w8_quantize_rows(x, ld, n, K, norm, eps, codes, ld_c, scales, None)


def product(codes=P, ld_c=112, scales=P, M=2, w=P, ld_w=112, ws=P, N=40, K=100, y=P, ld_y=40, yt=1, r=None, ld_r=0):
    return lib.glt_w8_linear_rows(codes, ld_c, scales, M, w, ld_w, ws, N, K, y, ld_y, yt, r, ld_r, None)


def linear(x=P, ld=100, M=2, norm=None, eps=1e-6, w=P, ld_w=112, ws=P, N=40, K=100, y=P, ld_y=40, yt=1, r=None, ld_r=0, space=P, n=BIG):
    return lib.glt_w8_linear(x, ld, M, norm, eps, w, ld_w, ws, N, K, y, ld_y, yt, r, ld_r, space, n, None)


def test_w8_rows():
    refused(rows(x=None), "null")
    refused(rows(scales=None), "null")
    refused(rows(ld=99), "rows")
    refused(rows(n=-1), "sizes")
    refused(rows(K=0), "sizes")
    refused(rows(K=131072, ld=131072, ld_c=131072), "sizes")
    refused(rows(codes=P + 8), "codes")
    refused(rows(ld_c=100), "codes")
    refused(rows(ld_c=96), "codes")
    for e in (-1e-6, float("nan"), float("inf")):
        refused(rows(norm=P, eps=e), "eps")
    assert rows(n=0, x=None, codes=None) == OK


@pytest.mark.parametrize("call", [product, linear])
def test_w8_products(call):
    refused(call(M=-1), "sizes")
    refused(call(N=0), "sizes")
    refused(call(K=131072), "sizes")
    refused(call(w=None), "w must")
    refused(call(w=P + 4), "w must")
    refused(call(ld_w=104), "w must")
    refused(call(ws=None), "null")
    refused(call(y=None), "rows of 40")
    refused(call(ld_y=39), "rows of 40")
    refused(call(r=P, ld_r=39), "rows of 40")
    refused(call(yt=2), "y_dtype")
    assert call(M=0) == OK
    refused(product(scales=None), "null")
    refused(product(codes=P + 1), "codes")
    need = C.c_int64()
    assert lib.glt_w8_linear_workspace(2, 100, C.byref(need)) == OK and need.value >= 2 * 112 + 8
    refused(linear(n=need.value - 1), "workspace")
    refused(linear(space=None), "workspace")
    refused(linear(space=P + 8), "workspace")
    refused(linear(x=None), "null")
    refused(linear(norm=P, eps=-1.0), "eps")
    refused(lib.glt_w8_linear_workspace(2, 100, None), "null")
    refused(lib.glt_w8_linear_workspace(2, 0, C.byref(need)), "sizes")


def test_w8_sizes_that_leave_32_bits_when_rounded_up():
    top = 2 ** 31 - 255
    refused(rows(n=top), "sizes")
    for call in (product, linear):
        refused(call(M=top), "sizes")
        refused(call(N=top, ld_y=top), "sizes")


# ---- the Python layer, on tensors that only say they lie on a GPU

BF16, I8 = torch.bfloat16, torch.int8


def w8(N=64, K=128, index=0):
    return serve.W8Weight(serve.W8Rows(on(torch.zeros(N, K, dtype=I8), index), on(torch.zeros(N), index)))


def test_weights_and_rows_of_another_kind(monkeypatch):
    host = Host(monkeypatch)
    c, s = torch.zeros(64, 128, dtype=I8), torch.zeros(64)
    for codes, scales in ((c, s), (on(c), s), (c, on(s)), (on(c.to(torch.uint8)), on(s)), (on(c), on(s.double())), (on(c[0]), on(s))):
        with pytest.raises(ValueError):
            serve.W8Weight.from_codes(codes, scales)
    for codes, scales in ((on(c), on(s[:3])), (on(torch.zeros(64, 100, dtype=I8)), on(s)), (on(torch.zeros(128, 64, dtype=I8).t()), on(s)),
                          (on(torch.zeros(0, 128, dtype=I8)), on(s[:0]))):
        with pytest.raises(ValueError):
            serve.W8Weight(serve.W8Rows(codes, scales))
    w = w8()
    x = on(torch.zeros(3, 128, dtype=BF16))
    for bad in (x.float(), on(torch.zeros(3, 127, dtype=BF16)), on(torch.zeros(128, 3, dtype=BF16).t()), torch.zeros(3, 128, dtype=BF16)):
        with pytest.raises(ValueError, match="x must"):
            w.linear(bad)
    for kw in (dict(norm=on(torch.zeros(127, dtype=BF16))), dict(norm=on(torch.zeros(128))), dict(norm=torch.zeros(128, dtype=BF16)),
               dict(resid=on(torch.zeros(3, 63, dtype=BF16))), dict(out=on(torch.zeros(2, 64, dtype=BF16))), dict(out_dtype=torch.float16)):
        with pytest.raises(ValueError):
            w.linear(x, **kw)
    with pytest.raises(ValueError, match="rows must"):
        w.linear_rows(serve.W8Rows(on(torch.zeros(3, 120, dtype=I8)), on(torch.zeros(3))))
    with pytest.raises(ValueError):
        serve.quantize_rows(torch.zeros(3, 128, dtype=BF16))
    with pytest.raises(ValueError):
        serve.quantize_rows(on(torch.zeros(3, 0, dtype=BF16)))
    assert not host.calls


def parts(index=0, other=None):
    def t(name, *shape, dtype=BF16):
        return on(torch.zeros(*shape, dtype=dtype), other if other is not None and name == "odd" else index)
    return t


def test_calls_run_on_their_tensors_device(monkeypatch):
    host = Host(monkeypatch)
    dev1 = dict(dtype=torch.int32)
    c = serve.Kv8Cache(8, 16, 2, 64, device="cuda:1")
    b = serve.Kv8Batch(on(torch.zeros(2, 4, **dev1), 1), on(torch.zeros(2, **dev1), 1), 2)
    p = serve.Kv8Prefix(on(torch.zeros(3, **dev1), 1), on(torch.zeros(1, **dev1), 1))
    q = on(torch.zeros(2, 4, 64, dtype=BF16), 1)
    x = on(torch.zeros(3, 128, dtype=BF16), 1)
    c.prefix_attention(b, p, q)
    c.attention(b, q, window=8, sinks=2)
    w8(index=1).linear(x)
    w8(index=1).linear_rows(serve.quantize_rows(x))
    assert host.calls and all(at == 1 for _, at, _ in host.calls) and host.current == 0
    names = [n for n, _, _ in host.calls]
    assert names == ["glt_kv8_prefix_attention", "glt_kv8_window_attention", "glt_w8_linear", "glt_w8_quantize_rows", "glt_w8_linear_rows"]


def test_operands_of_two_devices_are_refused(monkeypatch):
    host = Host(monkeypatch)
    i32 = dict(dtype=torch.int32)
    c, b = serve.Kv8Cache(8, 16, 2, 64), serve.Kv8Batch(on(torch.zeros(2, 4, **i32)), on(torch.zeros(2, **i32)), 2)
    q = on(torch.zeros(2, 4, 64, dtype=BF16))
    with pytest.raises(ValueError, match="cuda"):
        c.prefix_attention(b, serve.Kv8Prefix(on(torch.zeros(3, **i32), 1), on(torch.zeros(1, **i32), 1)), q)
    with pytest.raises(ValueError, match="device"):
        serve.Kv8Prefix(on(torch.zeros(3, **i32), 1), on(torch.zeros(1, **i32)))
    p = serve.Kv8Prefix(on(torch.zeros(3, **i32)), on(torch.zeros(1, **i32)))
    for bad in (on(torch.zeros(2, 4, 64, dtype=BF16), 1), on(torch.zeros(2, 4, 63, dtype=BF16)), on(torch.zeros(3, 4, 64, dtype=BF16))):
        with pytest.raises(ValueError):
            c.prefix_attention(b, p, bad)
    for ids, n in ((torch.zeros(3, dtype=torch.int64), torch.zeros(1, **i32)), (torch.zeros(3, 1, **i32), torch.zeros(1, **i32)),
                   (torch.zeros(3, **i32), torch.zeros(2, **i32)), (torch.zeros(3, **i32), torch.zeros((), **i32))):
        with pytest.raises(ValueError):
            serve.Kv8Prefix(on(ids), on(n))
    x = on(torch.zeros(3, 128, dtype=BF16))
    for kw in (dict(norm=on(torch.zeros(128, dtype=BF16), 1)), dict(resid=on(torch.zeros(3, 64, dtype=BF16), 1)),
               dict(out=on(torch.zeros(3, 64, dtype=BF16), 1))):
        with pytest.raises(ValueError, match="cuda:0"):
            w8().linear(x, **kw)
    with pytest.raises(ValueError):
        w8(index=1).linear(x)
    assert not host.calls


def test_calls_of_two_threads_and_captures_have_workspaces_of_their_own(monkeypatch):
    host = Host(monkeypatch)
    i32 = dict(dtype=torch.int32)
    c, b = serve.Kv8Cache(8, 16, 2, 64), serve.Kv8Batch(on(torch.zeros(2, 4, **i32)), on(torch.zeros(2, **i32)), 2)
    p = serve.Kv8Prefix(on(torch.zeros(3, **i32)), on(torch.zeros(1, **i32)))
    q, x, w = on(torch.zeros(2, 4, 64, dtype=BF16)), on(torch.zeros(3, 128, dtype=BF16)), w8()
    for name, call in (("glt_w8_linear", lambda: w.linear(x)), ("glt_kv8_prefix_attention", lambda: c.prefix_attention(b, p, q))):
        both = threading.Barrier(2)
        host.calls.clear()
        host.launched = lambda *_: both.wait(10) and 0
        threads = [threading.Thread(target=call) for _ in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        used = [args[-3] for n, _, args in host.calls if n == name]
        assert len(used) == 2 and used[0] != used[1]
        host.launched = lambda *_: 0
        host.calls.clear()
        kept, real = [], Host.empty
        with monkeypatch.context() as m:
            m.setattr(serve, "_capturing", lambda: True)
            m.setattr(host, "empty", lambda *a, **k: kept.append(real(host, *a, **k)) or kept[-1], raising=False)
            call()
            call()
        assert len({args[-3] for _, _, args in host.calls}) == 2


# ---- the decoder

@pytest.mark.parametrize("kw,word", [(dict(bits=3), "bits"), (dict(shared_tokens=-1), "negative"), (dict(window=-1), "negative"),
                                     (dict(sinks=2), "window"), (dict(window=8, shared_tokens=9), "prefix")])
def test_decoders(kw, word):
    with pytest.raises(ValueError, match=word):
        decode.Decoder(dict(), 4, 2, 64, 1, 8, **kw)


@pytest.mark.parametrize("ids", [torch.zeros(0, dtype=torch.int32), torch.zeros(11, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32),
                                 torch.zeros(3)])
def test_shared_prompts(ids):
    d = decode.Decoder.__new__(decode.Decoder)
    d.shared_tokens, d.held = 10, 0
    with pytest.raises(ValueError, match="shared"):
        d.share(ids)
    d.held = 1
    with pytest.raises(ValueError, match="hold"):
        d.share(torch.zeros(4, dtype=torch.int32))


@pytest.mark.parametrize("args", [["--shared", "-1"], ["--window", "9", "--shared", "9"], ["--sinks", "2"], ["--bits", "5"]])
def test_the_command(monkeypatch, args):
    monkeypatch.setattr(sys, "argv", ["decode"] + args)
    monkeypatch.setattr(decode, "random_weights", lambda **k: pytest.fail("weights were made"))
    with pytest.raises(SystemExit):
        decode.main()
