"""The operators captured where several workgroups join a sum in one launch, and called on two streams and by two threads at once.

In a file that runs last, behind the cooperative kernels' tests, as every test that uses a second stream.
"""
import threading

import pytest
import torch

from flashact_amd import attention, kv8, w4
from tests.test_gpu_attention import _qkv
from tests.test_gpu_kv8 import _filled, _ints

pytestmark = pytest.mark.gpu


def test_joined_parts_in_a_graph(gpu):
    """Up to four parts, joined by the last workgroup. A replay repeats the launch's number: the words that it leaves must not count."""
    q, k, v = _qkv(gpu, 1, 1000, 4000, 8, 1, 128, torch.bfloat16)
    i = torch.arange(1000, device=gpu)
    spans = torch.stack([torch.zeros_like(i), i + 3001], -1).to(torch.int32)
    assert attention._workspace_bytes(1, 1000, 4000, 8, 128) > 0
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = attention.attend(q, k, v, spans)
        z = attention.attend(y, k, v, spans)  # a second call in the first one's memory
    for n in range(6):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device=gpu))
        spans[:, 1] = (i + 3001 - 500 * n).clamp(min=0)
        g.replay()
        torch.cuda.synchronize()
        want = attention.attend(q, k, v, spans)
        assert torch.equal(y, want) and torch.equal(z, attention.attend(want, k, v, spans))


def test_two_graphs_of_one_pool(gpu):
    """Two captured steps that share their memory, replayed in turn: each finds the other's leftovers in its workspace."""
    cache, w = _filled(gpu, 3, 900, 1, 256, seed=4), w4.quantize(torch.randn(2048, 2048, device=gpu) * 0.02)
    wide = w4.quantize(torch.randn(2048, 16384, device=gpu) * 0.02)
    q, lens = torch.randn(3, 1, 8, 256, device=gpu).bfloat16(), _ints(gpu, 900, 450, 33)
    x = torch.randn(3, 16384, device=gpu).bfloat16()

    def one():
        return w4.linear(kv8.attend(q, cache, lens).view(3, 2048), w), w4.linear(x, wide)

    def two():
        return w4.linear(x, wide, out_dtype=torch.float32), kv8.attend(q, cache, lens)

    graphs, outs, pool = [], [], None
    for f in (one, two):
        f()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(f())
        pool = pool or g.pool()
        graphs.append(g)
    for n in range(6):
        q.copy_(torch.randn(q.shape, device=gpu))
        x.copy_(torch.randn(x.shape, device=gpu))
        lens.copy_(_ints(gpu, 900 - 100 * n, 20 + 90 * n, n))
        for g, out, f in zip(graphs, outs, (one, two)):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, f()))


def _calls(gpu):
    """Calls whose sums several workgroups join: by the last one, and by a second kernel."""
    cache = _filled(gpu, 2, 5000, 1, 256, seed=9)
    q, lens = torch.randn(2, 3, 8, 256, device=gpu).bfloat16(), _ints(gpu, 5000, 1200)
    few, k, v = _qkv(gpu, 1, 1024, 4096, 8, 1, 128, torch.float16)
    x, w = torch.randn(9, 16384, device=gpu).bfloat16(), w4.quantize(torch.randn(2048, 16384, device=gpu) * 0.02)
    return [lambda: kv8.attend(q, cache, lens), lambda: kv8.attend(q, cache, lens, causal=False, softcap=5.0),
            lambda: attention.attend(few, k, v), lambda: attention.attend(few[:, :64], k, v), lambda: w4.linear(x, w),
            lambda: w4.linear(x[:3], w)]


def test_two_streams_at_once(gpu):
    calls = _calls(gpu)
    refs = [f() for f in calls]
    streams, bad = [torch.cuda.Stream() for _ in range(2)], torch.zeros(2, dtype=torch.int64, device=gpu)
    torch.cuda.synchronize()
    for i in range(120):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                j = (i * (1 + 4 * n) + n) % len(calls)
                bad[n] += (calls[j]() != refs[j]).any()
    torch.cuda.synchronize()
    assert bad.tolist() == [0, 0]


def test_two_threads_at_once(gpu):
    calls = _calls(gpu)
    refs = [f() for f in calls]
    torch.cuda.synchronize()
    results, errors = {}, []

    def work(n):
        try:
            bad = torch.zeros((), dtype=torch.int64, device=gpu)
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(120):
                    j = (i * (1 + 4 * n) + n) % len(calls)
                    bad += (calls[j]() != refs[j]).any()
                torch.cuda.current_stream().synchronize()
            results[n] = bad.item()
        except Exception as e:  # reported by the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and results == {0: 0, 1: 0}
