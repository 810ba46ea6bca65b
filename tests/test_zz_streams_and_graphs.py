"""The operators on a stream of their own and in captured graphs, on the MI355X: every replay equals the eager result.

In a file that runs last: once a process that has made a cooperative launch begins to use a second stream, the runtime places
the workgroups of its later cooperative launches on the XCDs from another one on (FA_KSTATUS_XCD_MAP), and the cooperative
kernels' tests hold that status to be zero.
"""
import pytest
import torch

from flashact_amd import attention, kv8, prefill, w4
from tests.test_gpu_attention import _documents, _qkv
from tests.test_gpu_backbone import NL, _weights
from tests.test_gpu_kv8 import _filled, _ints

pytestmark = pytest.mark.gpu


def test_w4_streams_and_graphs(gpu):
    """On a stream of its own, and captured: every replay equals the eager result on the inputs of that time."""
    w = w4.quantize(torch.randn(64, 16384, device=gpu) * 0.02, 32)  # a split sum: two kernels and a workspace
    x = torch.randn(8, 16384, device=gpu).bfloat16()
    ref = w4.linear(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = w4.linear(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = w4.linear(x, w)
    for i in range(4):
        x.copy_(torch.randn(8, 16384, device=gpu))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, w4.linear(x, w))


def test_kv8_streams_and_graphs(gpu):
    cache = _filled(gpu, 2, 600, 2, 128, seed=6)
    q, lens = torch.randn(2, 3, 8, 128, device=gpu).bfloat16(), _ints(gpu, 600, 217)
    ref = kv8.attend(q, cache, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = kv8.attend(q, cache, lens)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, ref)
    # a captured step: store a token, attend, the length grows between replays
    k, v = (torch.randn(2, 1, 2, 128, device=gpu).bfloat16() for _ in range(2))
    start, qs = _ints(gpu, 300, 217), q[:, :1].contiguous()
    copies = [{n: t.clone() for n, t in cache.items()} for _ in range(2)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kv8.store(copies[0], k, v, start)
        y = kv8.attend(qs, copies[0], start + 1)
    for i in range(5):
        k.copy_(torch.randn(2, 1, 2, 128, device=gpu))
        qs.copy_(torch.randn(2, 1, 8, 128, device=gpu))
        g.replay()
        torch.cuda.synchronize()
        kv8.store(copies[1], k, v, start)
        assert torch.equal(y, kv8.attend(qs, copies[1], start + 1))
        assert all(torch.equal(copies[0][n], copies[1][n]) for n in cache)
        start += 1


def test_attention_streams_and_graphs(gpu):
    q, k, v = _qkv(gpu, 1, 200, 200, 4, 2, 128, torch.bfloat16)
    spans = _documents(gpu, [120, 80], [50, 80])
    ref = attention.attend(q, k, v, spans)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = attention.attend(q, k, v, spans)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = attention.attend(q, k, v, spans)
    for i in range(4):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device=gpu))
        spans.copy_(_documents(gpu, [60 + 30 * i, 140 - 30 * i], [10 * i, 140 - 30 * i]))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, attention.attend(q, k, v, spans))


def test_extend_in_a_graph(gpu):
    """One captured step answers token after token: its replays equal the eager steps on a copy of the cache."""
    _, _, w4s, ln = _weights(gpu, seed=1)
    caches = [kv8.make_caches(NL, 3, 64, device=gpu) for _ in range(2)]
    lens, x = _ints(gpu, 0, 5, 29), torch.randn(3, 1, 2048, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm-up on a third cache: library handles are made outside the capture
        prefill.extend(w4s, *ln, x, kv8.make_caches(NL, 3, 64, device=gpu), lens)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = prefill.extend(w4s, *ln, x, caches[0], lens)
    for _ in range(5):
        x.copy_(torch.randn(3, 1, 2048, device=gpu))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, prefill.extend(w4s, *ln, x, caches[1], lens))
        for a, b in zip(*caches):
            assert all(torch.equal(a[n], b[n]) for n in a)
        lens += 1


def test_attention_parts_in_a_graph(gpu):
    """Few queries over many keys, two kernels and a workspace: every replay equals the eager result on the inputs of that time."""
    q, k, v = _qkv(gpu, 1, 20, 9000, 4, 2, 128, torch.bfloat16)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = attention.attend(q, k, v)
    for i in range(4):
        q.copy_(torch.randn(1, 20, 4, 128, device=gpu))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, attention.attend(q, k, v))
