"""Decoding and scoring calls from several host threads, streams and captured graphs."""
import threading

import pytest
import torch

from glt_b200 import serve

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_two_threads_share_a_weight_a_cache_and_a_stream():
    """Each thread's results are those of its calls alone."""
    g = torch.Generator(device=DEV).manual_seed(0)
    w = serve.W4Weight.quantize((torch.randn(512, 1024, device=DEV, generator=g) * 0.1).to(torch.bfloat16), 64)
    cache = serve.Kv8Cache(80, 32, 2, 64)
    table = torch.arange(80, device=DEV, dtype=torch.int32).view(4, 20)
    kv = torch.randn(2, 2400, 2, 64, device=DEV, generator=g).to(torch.bfloat16)
    cache.append(serve.Kv8Batch(table, torch.zeros(4, device=DEV, dtype=torch.int32), 2400), kv[0], kv[1])

    def inputs(rows, tokens):
        batch = serve.Kv8Batch(table, torch.full((4,), tokens - 1, device=DEV, dtype=torch.int32), 4)
        return (torch.randn(rows, 1024, device=DEV, generator=g).to(torch.bfloat16), batch,
                torch.randn(4, 8, 64, device=DEV, generator=g).to(torch.bfloat16))

    def results(x, batch, q):
        return (w.linear(x), *cache.attention(batch, q))

    jobs = [inputs(20, 600), inputs(27, 431)]
    want = [results(*j) for j in jobs]
    torch.cuda.synchronize()
    got, ready = [None, None], threading.Barrier(2)

    def run(i):
        ready.wait(30)
        got[i] = [results(*jobs[i]) for _ in range(300)]

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))
