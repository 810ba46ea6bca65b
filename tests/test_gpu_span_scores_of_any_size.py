"""attention.attend whose scores are far past 2^22, on the MI355X: the best key's value comes back as it is (test_gpu_scores_of_any_size)."""
import pytest
import torch

from flashact_amd import attention
from tests import span_case
from tests.test_gpu_scores_of_any_size import DTYPES, SIZES, _inputs, _lead, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("tokens,heads,kv_heads,hd,n", [(1, 8, 1, 256, 300), (3, 6, 2, 128, 700), (70, 4, 4, 96, 700), (300, 8, 2, 128, 1100),
                                                        (130, 2, 1, 256, 900), (513, 4, 4, 64, 600), (1, 2, 1, 72, 9000)])
@pytest.mark.parametrize("sign", [1, -1])
def test_spans(gpu, dtype, sizes, tokens, heads, kv_heads, hd, n, sign):
    for best in (3, n // 2):
        q, k, v = _inputs(gpu, dtype, sizes, tokens, heads, kv_heads, hd, n, best, sign)
        _lead(q, k, best, hd ** -0.5)
        want = _want(v, best, heads, tokens)
        assert torch.equal(attention.attend(q, k, v), want)
        assert torch.equal(attention.attend(q, k, v, slopes=torch.full((heads,), 0.5, device=gpu)), want)
        cap = 8.0 * float(q.abs().amax()) * float(k.abs().amax()) * hd ** 0.5
        assert torch.equal(attention.attend(q, k, v, softcap=cap), want)
        last = torch.tensor([[0, n - 5]], dtype=torch.int32, device=gpu).expand(tokens, 2).contiguous()
        assert torch.equal(attention.attend(q, k, v, last), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,heads,kv_heads,hd,n", [(3, 6, 2, 128, 700), (70, 4, 4, 96, 700), (300, 8, 2, 128, 1100), (130, 2, 1, 256, 900)])
def test_large_scores_of_other_rows_change_nothing(gpu, dtype, tokens, heads, kv_heads, hd, n):
    """Every other token's queries are small enough for ordinary scores: their results are those of a call without the large ones."""
    q, k, v = _inputs(gpu, dtype, (8000.0, 10000.0), tokens, heads, kv_heads, hd, n, 7, 1)
    q[:, ::2] *= 2.0 ** -27 if dtype is torch.bfloat16 else 2.0 ** -24
    alone = q.clone()
    alone[:, 1::2] = 0
    both, one = attention.attend(q, k, v), attention.attend(alone, k, v)
    assert torch.equal(both[:, ::2], one[:, ::2])
    span_case.check(one, *span_case.attend(alone, k, v))
