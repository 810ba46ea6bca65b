"""Calls of the operators for many requests that their documentation allows and that are rarely made."""
import pytest
import torch

from flashact_amd import lora, paged, tokens
from tests import kv8_case, paged_case as C, tokens_case
from tests.lora_case import make
from tests.test_gpu_paged import _ints

pytestmark = pytest.mark.gpu


def test_pages(gpu):
    pool, table = C.filled(gpu, (700, 45), 1, 128, torch.bfloat16, seed=1, width=4100)
    wide = torch.randn(2, 40, 3, 8, 128, device=gpu).bfloat16()
    q, lens = wide[:, :, 1], _ints(gpu, 700, 45)  # two tiles a wave, queries of any stride
    k, v = C.rows_of(pool, table[:, :22])
    ref = paged.attend(q, pool, table, lens)
    kv8_case.check(ref, *kv8_case.attend(q, k, v, (700, 45)))
    out = torch.empty_like(ref)
    assert paged.attend(q, pool, table, lens, out=out) is out and torch.equal(out, ref)
    assert not paged.attend(q, pool, table, lens, count=_ints(gpu, 0, 0)).any()
    none = torch.empty(2, 0, 8, 128, device=gpu, dtype=torch.bfloat16)
    assert paged.attend(none, pool, table, lens, out=none) is none
    before = {m: t.clone() for m, t in pool.items()}
    rows = torch.randn(2, 3, 1, 128, device=gpu).bfloat16()
    assert not paged.append(pool, table, rows, rows, lens, _ints(gpu, 0, -4), q=q[:, :3], freqs=paged.frequencies(128, device=gpu)).any()
    assert paged.append(pool, table, rows[:, :0], rows[:, :0], lens) is None
    k0, v0 = paged.load(pool, table[:, :22], lens, k=rows[:, :0], v=rows[:, :0])
    assert k0.shape == v0.shape == (2, 0, 1, 128)
    assert all(torch.equal(pool[m], before[m]) for m in "kv")
    one = rows[:, :, :, :1].expand(2, 3, 1, 128).contiguous()[:, :1].expand(2, 3, 1, 128)  # one row for all tokens
    paged.append(pool, table, one, one, lens)
    got, _ = paged.load(pool, table[:, :24], _ints(gpu, 703, 48))
    for b, n in enumerate((700, 45)):
        assert torch.equal(got[b, n:n + 3], one[b])


def test_adapters(gpu):
    gen = torch.Generator(device=gpu).manual_seed(4)
    y, x, bank = make(gen, gpu, 3, 16, 64, 136, torch.float16, 1100, torch.float32)
    index = (torch.arange(1100, device=gpu) // 90 % 4 - 1).int()
    ref = lora.add(y, x, bank, index, gate="gelu")
    out = torch.empty_like(ref)
    assert lora.add(y, x, bank, index, gate="gelu", out=out) is out and torch.equal(out, ref)
    wide = torch.full((1100, 200), float("nan"), device=gpu, dtype=torch.float16)
    wide[:, 8:144] = x
    assert torch.equal(lora.add(y, wide[:, 8:144], bank, index, gate="gelu"), ref)
    # the same rows alone: tiles begin elsewhere, adapters meet in other pairs
    assert torch.equal(lora.add(y[7:300], x[7:300].contiguous(), bank, index[7:300].contiguous(), gate="gelu"), ref[7:300])


def test_tokens(gpu):
    x = torch.randn(3, 5, 777, device=gpu).half()
    t = torch.randint(0, 777, (3, 5), device=gpu)
    got, flat = tokens.logprobs(x, t, top=4), tokens.logprobs(x.view(15, 777), t.view(15).int(), top=4)
    for a, b in zip(got, flat):
        assert a.shape[:2] == (3, 5) and torch.equal(a.reshape(b.shape), b)
    ref, _ = tokens_case.logprobs(x.view(15, 777).double(), t.view(15), 4)
    assert torch.equal(flat.top_tokens.long(), ref["top_tokens"].to(gpu))
    one = x[:1, :1, :].expand(1, 6, 777).reshape(6, 777)[:, :1]  # a vocabulary of one
    r = tokens.logprobs(one, torch.zeros(6, dtype=torch.int64, device=gpu), top=1)
    assert not r.logprob.any() and not r.entropy.any() and not r.top_tokens.any()
    same = tokens.logprobs(x[0, :1].expand(4, 777), t[0, :4])  # one row read four times
    assert torch.equal(same.entropy, same.entropy[:1].expand(4))
