"""What the backbone's paths for many requests allow at their edges: no tokens, empty prompts, tables that end, one request's pages given
back and used by another."""
import pytest
import torch

from flashact_amd import paged, prefill
from tests.test_gpu_backbone import NL, _ints, _weights
from tests.test_gpu_requests import _Reference, _banks, _close

pytestmark = pytest.mark.gpu


def test_no_tokens_and_empty_prompts(gpu):
    _, packed, w4s, ln = _weights(gpu, seed=2)
    banks = _banks(gpu, 5)
    adapters = (banks, _ints(gpu, 1, 0, 1))
    pools, table = paged.make_pools(NL, 6, device=gpu), _ints(gpu, 0, 1, 2, 3, 4, 5).view(3, 2)
    x = torch.randn(20, 2048, device=gpu)
    out = prefill.prefill_packed(packed, *ln, x, [0, 20, 0], pools, table=table, adapters=adapters)
    ref = _Reference(packed, ln, banks, 0)
    _close(out, ref.run(x, prefix=20), x)
    before = [{m: t.clone() for m, t in p.items()} for p in pools]
    assert prefill.prefill_packed(packed, *ln, x[:0], [0, 0, 0], pools, table=table, adapters=adapters).shape == (0, 2048)
    assert prefill.extend(w4s, *ln, x[:0].view(3, 0, 2048), pools, _ints(gpu, 0, 20, 0), table=table, adapters=adapters).shape == (3, 0, 2048)
    assert all(torch.equal(a[m], b[m]) for a, b in zip(pools, before) for m in "kv")
    new = torch.randn(3, 2, 2048, device=gpu)  # two requests begin with these tokens, one goes on
    out = prefill.extend(w4s, *ln, new, pools, _ints(gpu, 0, 20, 0), table=table, adapters=adapters)
    _close(out[1], ref.run(new[1]), new[1])
    for b in (0, 2):
        _close(out[b], _Reference(packed, ln, banks, 1).run(new[b]), new[b])
    head = torch.randn(100, 2048, device=gpu).bfloat16()
    assert prefill.answer(head, ln[0][0], out[:, :0]).top_tokens.shape == (3, 0, 1)


def test_tokens_behind_the_tables_end_are_not_real(gpu):
    _, packed, w4s, ln = _weights(gpu, seed=2)
    pools, table = paged.make_pools(NL, 4, device=gpu), _ints(gpu, 2, 0).view(1, 2)
    x = torch.randn(62, 2048, device=gpu)
    prefill.prefill_packed(packed, *ln, x, [62], pools, table=table)
    ref = _Reference(packed, ln, [{}] * NL, -1)
    ref.run(x, prefix=62)
    new = torch.randn(1, 5, 2048, device=gpu)
    out = prefill.extend(w4s, *ln, new, pools, _ints(gpu, 62), table=table)
    _close(out[0, :2], ref.run(new[0, :2]), new[0, :2])
    for p in pools:
        assert not p["k"][[1, 3]].any() and not p["v"][[1, 3]].any()


def test_pages_given_back(gpu):
    """A request's pages, full of another's rows, serve the next one."""
    _, packed, w4s, ln = _weights(gpu, seed=3)
    pools = paged.make_pools(NL, 3, device=gpu)
    table = _ints(gpu, 1, 0, 2).view(1, 3)
    prefill.prefill_packed(packed, *ln, torch.full((96, 2048), 1e4, device=gpu), [96], pools, table=table)
    x, new = torch.randn(40, 2048, device=gpu), torch.randn(1, 1, 2048, device=gpu)
    table = table.flip(1).contiguous()
    prefill.prefill_packed(packed, *ln, x, [40], pools, table=table)
    ref = _Reference(packed, ln, [{}] * NL, -1)
    ref.run(x, prefix=40)
    _close(prefill.extend(w4s, *ln, new, pools, _ints(gpu, 40), table=table)[0], ref.run(new[0]), new[0])
