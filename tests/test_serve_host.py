"""The host side of the decoding and scoring calls, without a GPU."""
import threading

import pytest
import torch

from glt_b200 import serve
from glt_b200._lib import GltError
from serve_host import Host, on


def weight(N=64, K=128, group=32, index=0):
    need = serve.C.c_int64()
    serve.check(serve.lib.glt_w4_packed_bytes(N, K, group, 0, serve.C.byref(need)))
    return serve.W4Weight(on(torch.zeros(need.value, dtype=torch.uint8), index), N, K, group, False)


def cache_and_batch(seqs=2, new=1):
    cache = serve.Kv8Cache(8, 16, 2, 64)
    table = on(torch.zeros(seqs, 4, dtype=torch.int32))
    return cache, serve.Kv8Batch(table, on(torch.zeros(seqs, dtype=torch.int32)), seqs * new)


def test_calls_of_two_threads_have_workspaces_of_their_own(monkeypatch):
    """A call is up to two launches that share a workspace, and two threads' launches on a stream may
    come in any order: neither may use the other's."""
    host = Host(monkeypatch)
    w = weight()
    cache, batch = cache_and_batch()
    x, q = on(torch.zeros(20, 128, dtype=torch.bfloat16)), on(torch.zeros(2, 4, 64, dtype=torch.bfloat16))
    for name, at, call in (("glt_w4_linear", -3, lambda: w.linear(x)),
                           ("glt_kv8_attention", -3, lambda: cache.attention(batch, q))):
        both = threading.Barrier(2)
        host.calls.clear()
        host.launched = lambda *_: both.wait(10) and 0    # both calls are under way at once
        threads = [threading.Thread(target=call) for _ in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        used = [args[at] for n, _, args in host.calls if n == name]
        assert len(used) == 2 and used[0] != used[1]


def test_objects_share_a_workspace_for_each_stream(monkeypatch):
    """One thread's calls on a stream run in order: its weights and caches need one workspace, not one each."""
    host = Host(monkeypatch)
    x = on(torch.zeros(20, 128, dtype=torch.bfloat16))
    for w in (weight(), weight(), weight()):
        w.linear(x)
    first = {args[-3] for _, _, args in host.calls}
    host.stream = 64
    weight().linear(x)
    assert len(first) == 1 and host.calls[-1][2][-3] not in first


def test_calls_under_capture_have_workspaces_of_their_own(monkeypatch):
    """Graphs may replay side by side, so none may hold the stream's workspace."""
    host = Host(monkeypatch)
    w, x = weight(), on(torch.zeros(20, 128, dtype=torch.bfloat16))
    w.linear(x)
    monkeypatch.setattr(serve, "_capturing", lambda: True)
    kept = []
    real = host.empty
    monkeypatch.setattr(host, "empty", lambda *a, **k: kept.append(real(*a, **k)) or kept[-1], raising=False)
    w.linear(x)
    w.linear(x)
    assert len({args[-3] for _, _, args in host.calls}) == 3


def test_weights_of_host_memory_are_refused(monkeypatch):
    """Codes, scales and zeros as a checkpoint's reader returns them: the kernel would follow host addresses."""
    host = Host(monkeypatch)
    parts = (torch.zeros(64, 128, dtype=torch.uint8), torch.zeros(64, 4, dtype=torch.bfloat16),
             torch.zeros(64, 4, dtype=torch.uint8))
    for i in range(3):
        mixed = [t if i == j else on(t) for j, t in enumerate(parts)]
        with pytest.raises(ValueError, match="CUDA"):
            serve.W4Weight.from_codes(*mixed)
    with pytest.raises(ValueError, match="CUDA"):
        serve.W4Weight.from_codes(*parts[:2])
    assert not host.calls


@pytest.mark.parametrize("packed", [lambda n: torch.zeros(n, dtype=torch.uint8), lambda n: on(torch.zeros(n - 1, dtype=torch.uint8)),
                                    lambda n: on(torch.zeros(n, dtype=torch.int8)), lambda n: on(torch.zeros(2 * n, dtype=torch.uint8)[::2])])
def test_packed_weights_that_do_not_hold_the_matrix_are_refused(monkeypatch, packed):
    """Every read of `linear` and `unpack` lies within the size that N, K and the group ask for."""
    Host(monkeypatch)
    need = serve.C.c_int64()
    serve.check(serve.lib.glt_w4_packed_bytes(64, 128, 32, 0, serve.C.byref(need)))
    with pytest.raises(ValueError, match="packed"):
        serve.W4Weight(packed(need.value), 64, 128, 32, False)


@pytest.mark.parametrize("group", [0, -32, 48, 256])
def test_groups_that_do_not_fit_are_refused_before_any_launch(monkeypatch, group):
    host = Host(monkeypatch)
    with pytest.raises(GltError):
        serve.quantize_w4(on(torch.zeros(4, 128, dtype=torch.bfloat16)), group)
    assert not host.calls


def calls(index, other=None):
    """Every call of the module, its tensors on device `index`; with `other`, one call for each operand
    that could lie elsewhere, and there it does: (name, call)."""
    def t(name, *shape, dtype=torch.bfloat16):
        return lambda at: on(torch.zeros(*shape, dtype=dtype), other if at == name else index)

    i32, u8, f32 = torch.int32, torch.uint8, torch.float32
    table, lengths = t("block_table", 2, 4, dtype=i32), t("lengths", 2, dtype=i32)
    starts, start = t("row_start", 3, dtype=i32), t("start", 2, dtype=i32)
    k, v, q, out = t("k", 2, 2, 64), t("v", 2, 2, 64), t("q", 2, 4, 64), t("out", 2, 4, 64)
    pools = [t(n, 8, 2, 16, 64, dtype=u8) for n in ("pool k", "pool v")]
    scales = [t(n, 8, 2, dtype=f32) for n in ("k_scale", "v_scale")]
    mask = t("token_mask", 2, 64, dtype=u8)
    codes, sc, zeros = t("codes", 64, 128, dtype=u8), t("scales", 64, 4), t("zeros", 64, 4, dtype=u8)
    x, resid, y = t("x", 20, 128), t("resid", 20, 64), t("y", 20, 64)
    logits, targets, d, dout = t("logits", 3, 50), t("targets", 3, dtype=i32), t("d_logp", 3, dtype=f32), t("dlogits", 3, 50)
    de = t("d_entropy", 3, dtype=f32)

    def cache(at):
        return serve.Kv8Cache.from_buffers(*(p(at) for p in pools + scales))

    def batch(at):
        return serve.Kv8Batch(table(at), lengths(at), 2, row_start=starts(at))

    def scores(at):
        return serve.token_logprobs(logits(at), targets(at), top=2)

    def gradient(at):
        f = scores(None)
        return serve.token_logprobs_bwd(logits(at), targets(at), f, d(at), de(at), out=dout(at))

    w = {  # call: the operands that it takes
        "append": (lambda at: cache(at).append(batch(at), k(at), v(at)),
                   ("block_table", "lengths", "row_start", "pool k", "pool v", "k_scale", "v_scale", "k", "v")),
        "attention": (lambda at: cache(None).attention(batch(None), q(at), token_mask=mask(at), out=out(at)),
                      ("q", "token_mask", "out")),
        "read": (lambda at: cache(None).read(batch(None), start(at), 3), ("start",)),
        "from_codes": (lambda at: serve.W4Weight.from_codes(codes(at), sc(at), zeros(at)), ("codes", "scales", "zeros")),
        "quantize": (lambda at: serve.quantize_w4(x(at), 32, True), ()),
        "unpack": (lambda at: serve.W4Weight.from_codes(codes(None), sc(None)).unpack(), ()),
        "linear": (lambda at: serve.W4Weight.from_codes(codes(None), sc(None)).linear(x(at), resid(at), out=y(at)),
                   ("x", "resid", "y")),
        "token_logprobs": (scores, ("logits", "targets")),
        "token_logprobs_bwd": (gradient, ("logits", "targets", "d_logp", "d_entropy", "dlogits")),
    }
    if other is None:
        return [(name, lambda f=f: f(None)) for name, (f, _) in w.items()]
    return [(f"{name}: {o}", lambda f=f, o=o: f(o)) for name, (f, ops) in w.items() for o in ops]


def test_calls_run_on_their_tensors_device(monkeypatch):
    """A launch goes to the device that is current, and so do its grid and its error word."""
    host = Host(monkeypatch)
    for index in (0, 1):
        for name, call in calls(index):
            for current in (0, 1):
                host.current = current
                host.calls.clear()
                call()
                assert host.calls and {at for _, at, _ in host.calls} == {index}, name
                assert host.current == current, name


def test_operands_of_two_devices_are_refused(monkeypatch):
    host = Host(monkeypatch)
    for name, call in calls(0, other=1):
        before = len(host.calls)
        with pytest.raises(ValueError):
            call()
            pytest.fail(name)
        assert all(n == "glt_w4_pack" or n == "glt_token_logprobs" for n, _, _ in host.calls[before:]), name


def test_workspaces_follow_the_device(monkeypatch):
    """The default stream has the same handle on every device."""
    host = Host(monkeypatch)
    x = [on(torch.zeros(20, 128, dtype=torch.bfloat16), i) for i in (0, 1)]
    w = [weight(index=i) for i in (0, 1)]
    for i in (0, 1, 0, 1):
        host.current = i
        w[i].linear(x[i])
    at = [args[-3] for _, _, args in host.calls]
    assert at[0] == at[2] != at[1] == at[3]


def test_a_decoder_steps_on_its_own_device(monkeypatch):
    from glt_b200 import decode
    host = Host(monkeypatch)
    d = decode.Decoder.__new__(decode.Decoder)
    d.embed = on(torch.zeros(4, 64), 1)
    d.seqs, d.max_tokens, d.held = 1, 4, 0
    d._step = lambda ids: host.current
    assert d.step(torch.zeros(1, 1, dtype=torch.int32)) == 1 and host.current == 0
