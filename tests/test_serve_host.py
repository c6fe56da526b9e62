"""The host side of the decoding and scoring calls, without a GPU."""
import threading

import pytest
import torch

from glt_b200 import serve
from glt_b200._lib import GltError
from serve_host import Host, on


def weight(N=64, K=128, group=32):
    need = serve.C.c_int64()
    serve.check(serve.lib.glt_w4_packed_bytes(N, K, group, 0, serve.C.byref(need)))
    return serve.W4Weight(on(torch.zeros(need.value, dtype=torch.uint8)), N, K, group, False)


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
