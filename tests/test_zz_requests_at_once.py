"""The operators of many requests captured, on a stream of their own, and called on two streams and by two threads at once.

In a file that runs last, behind the cooperative kernels' tests, as every test that uses a second stream.
"""
import threading

import pytest
import torch

from flashact_amd import lora, paged, prefill, tokens
from tests.test_gpu_backbone import NL, _ints, _weights
from tests.test_gpu_requests import _banks

pytestmark = pytest.mark.gpu


def _pool(gpu, pages, heads, hd, seed=0):
    gen = torch.Generator(device=gpu).manual_seed(seed)
    pool = paged.make_pools(1, pages, heads, hd, device=gpu)[0]
    for t in pool.values():
        t.copy_(torch.randn(t.shape, generator=gen, device=gpu))
    return pool


def _table(gpu, samples, width, pages, seed=0):
    return torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:samples * width].view(samples, width).int().to(gpu)


def _bank(gpu, n, k, rank, adapters=3):
    return lora.pack([(torch.randn(rank, k, device=gpu) * k ** -0.5, torch.randn(n, rank, device=gpu) * 0.1, 1.0) for _ in range(adapters)])


def test_a_step_of_all_of_them_in_a_graph(gpu):
    """A captured step: rows in, attention, an adapter, log probabilities, all with sums that several workgroups join. Every replay equals
    the eager step on a copy of the pool, with other lengths, tables and adapters each time."""
    b, width = 5, 40
    pools = [_pool(gpu, 300, 2, 128, seed=1) for _ in range(2)]
    table, lens = _table(gpu, b, width, 300), _ints(gpu, 1, 1200, 31, 0, 640)
    freqs, bank = paged.frequencies(64, device=gpu), _bank(gpu, 50007, 1024, 16)
    k, v, q = (torch.randn(b, 1, h, 128, device=gpu).bfloat16() for h in (2, 2, 8))
    base, index, token = torch.randn(b, 50007, device=gpu), _ints(gpu, 0, 2, -1, 1, 0), torch.arange(b, device=gpu)

    def step(pool):
        turned = paged.append(pool, table, k, v, lens, q=q, freqs=freqs)
        o = paged.attend(turned, pool, table, lens + 1)
        y = lora.add(base, o.view(b, 1024), bank, index)
        return o, y, *tokens.logprobs(y, token, top=5, scale=0.7)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(pools[0])
    for n in range(6):
        for x in (k, v, q, base):
            x.copy_(torch.randn(x.shape, device=gpu))
        if n % 2:
            table.copy_(_table(gpu, b, width, 300, seed=n))
            index.copy_(_ints(gpu, 2 - n % 3, -1, n % 3, 0, 1))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, step(pools[1])))
        assert all(torch.equal(pools[0][m], pools[1][m]) for m in "kv")
        lens.add_(1)
        token.add_(10007)


def test_two_graphs_of_one_pool_of_memory(gpu):
    """Two captured steps that share their memory, replayed in turn: each finds the other's leftovers in its workspaces."""
    pool, table = _pool(gpu, 400, 1, 256), _table(gpu, 3, 100, 400)
    q, lens = torch.randn(3, 1, 8, 256, device=gpu).bfloat16(), _ints(gpu, 3200, 450, 33)
    logits, token = torch.randn(3, 130001, device=gpu), _ints(gpu, 5, 130000, 77)
    bank, x, y, index = _bank(gpu, 2048, 16384, 8), torch.randn(3, 16384, device=gpu).bfloat16(), torch.randn(3, 2048, device=gpu), _ints(gpu, 0, 1, 1)

    def one():
        r = tokens.logprobs(logits, token, top=8)
        return paged.attend(q, pool, table, lens), r.logprob, r.entropy, r.top_tokens, lora.add(y, x, bank, index)

    def two():
        return lora.add(y, x, bank, index), paged.attend(q, pool, table, lens), *tokens.logprobs(logits, token, top=2)

    graphs, outs, memory = [], [], None
    for f in (one, two):
        f()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=memory):
            outs.append(f())
        memory = memory or g.pool()
        graphs.append(g)
    for n in range(6):
        for t in (q, logits, x, y):
            t.copy_(torch.randn(t.shape, device=gpu))
        lens.copy_(_ints(gpu, 3200 - 500 * n, 20 + 90 * n, n))
        for g, out, f in zip(graphs, outs, (one, two)):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, f()))


def test_extend_with_pages_and_adapters_in_a_graph(gpu):
    """One captured step of the backbone answers token after token; in between the requests change pages and adapters."""
    _, _, w4s, ln = _weights(gpu, seed=1)
    pools = [paged.make_pools(NL, 12, device=gpu) for _ in range(2)]
    tables = [_table(gpu, 3, 4, 12, seed=i) for i in range(2)]
    table, lens, x = tables[0].clone(), _ints(gpu, 0, 5, 29), torch.randn(3, 1, 2048, device=gpu)
    adapters = _banks(gpu, 2), _ints(gpu, 1, 0, -1)
    head = torch.randn(4001, 2048, device=gpu).bfloat16() * 0.05

    def step(pool):
        y = prefill.extend(w4s, *ln, x, pool, lens, table=table, adapters=adapters)
        return y, *prefill.answer(head, ln[0][0], y, top=3)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm-up on other pools: library handles are made outside the capture
        step(paged.make_pools(NL, 12, device=gpu))
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(pools[0])
    for n in range(6):
        x.copy_(torch.randn(3, 1, 2048, device=gpu))
        if n == 3:
            table.copy_(tables[1])
            lens.copy_(_ints(gpu, 0, 0, 0))
            adapters[1].copy_(_ints(gpu, -1, 1, 0))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(pools[1])))
        for a, b in zip(*pools):
            assert all(torch.equal(a[m], b[m]) for m in a)
        lens += 1


def _calls(gpu):
    """Calls with workspaces; each returns one tensor."""
    pool, table = _pool(gpu, 500, 1, 256, seed=9), _table(gpu, 2, 200, 500)
    q, lens = torch.randn(2, 3, 8, 256, device=gpu).bfloat16(), _ints(gpu, 5000, 1200)
    logits, token = torch.randn(2, 200003, device=gpu), _ints(gpu, 9, 200000)
    bank, x, y = _bank(gpu, 2048, 4096, 24), torch.randn(70, 4096, device=gpu).bfloat16(), torch.randn(70, 2048, device=gpu)
    index = (torch.arange(70, device=gpu) % 4 - 1).int()
    return [lambda: paged.attend(q, pool, table, lens), lambda: paged.attend(q, pool, table, lens, causal=False, softcap=5.0),
            lambda: tokens.logprobs(logits, token, top=4).top_logprobs, lambda: tokens.logprobs(logits, token).entropy,
            lambda: lora.add(y, x, bank, index), lambda: lora.add(y[:3], x[:3], bank, index[:3]),
            lambda: paged.load(pool, table, lens)[0]]


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
