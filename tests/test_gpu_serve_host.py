"""Decoding and scoring calls from several host threads, streams and captured graphs."""
import os
import subprocess
import sys
import threading

import pytest
import torch

from glt_b200 import serve

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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


FIRST = """
import sys, torch
from glt_b200 import serve
g = torch.Generator(device="cuda").manual_seed(0)
call = sys.argv[1]
if call == "linear":
    codes = torch.randint(0, 16, (256, 512), device="cuda", generator=g).to(torch.uint8)
    w = serve.W4Weight.from_codes(codes, torch.rand(256, 16, device="cuda", generator=g).to(torch.bfloat16))
    x = torch.randn(int(sys.argv[2]), 512, device="cuda", generator=g).to(torch.bfloat16)
    run = lambda: (w.linear(x),)
elif call == "token_logprobs":
    x = torch.randn(3, 5000, device="cuda", generator=g)
    run = lambda: serve.token_logprobs(x, top=3)[1:5]
else:
    cache = serve.Kv8Cache(8, 32, 2, 64)
    batch = serve.Kv8Batch(torch.arange(8, device="cuda", dtype=torch.int32).view(2, 4),
                           torch.zeros(2, device="cuda", dtype=torch.int32), 80)
    k, v, q = (torch.randn(80, n, 64, device="cuda", generator=g).to(torch.bfloat16) for n in (2, 2, 8))
    def run():
        cache.append(batch, k, v)
        return cache.attention(batch, q)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
graph.replay()
torch.cuda.synchronize()
for a, b in zip(got, run()):
    assert torch.equal(a, b)
print("same")
"""


@pytest.mark.parametrize("call", [["linear", "1"], ["linear", "20"], ["token_logprobs"], ["attention"]])
def test_a_process_s_first_call_may_be_captured(call):
    """No call allocates, the first one on a device included: memory allocated under capture invalidates it."""
    p = subprocess.run([sys.executable, "-c", FIRST, *call], capture_output=True, text=True, timeout=120, cwd=ROOT)
    assert p.returncode == 0 and p.stdout.strip() == "same", p.stderr[-600:]
