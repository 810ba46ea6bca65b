"""Edges of ``attention.attend`` on the MI355X: a scale of zero, caps, weights far below the largest."""
import math

import pytest
import torch

from flashact_amd import attention
from tests import span_case as C
from tests.test_gpu_attention import DTYPES, _qkv, _spans

pytestmark = pytest.mark.gpu


ZERO = [
    # b, tq, tk, heads, kv_heads, hd, spans
    (1, 130, 130, 2, 1, 128, "causal"),
    (2, 100, 100, 2, 2, 96, "random"),         # empty, reversed and single-key spans
    (1, 70, 77, 2, 1, 64, None),               # no spans, the last tile of keys is not whole
    (1, 1500, 1500, 48, 16, 128, "documents"),
    (1, 64, 9001, 8, 1, 256, "causal"),        # parts, joined by a kernel
    (1, 1000, 4000, 8, 2, 64, "random"),       # parts, joined by the last workgroup
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ZERO, ids=lambda c: "-".join(str(x) for x in c))
def test_a_scale_of_zero_gives_the_mean(gpu, case, dtype):
    """Every score is zero: a query gets the mean of the values that it sees, one that sees none zeros."""
    b, tq, tk, h, hkv, hd, kind = case
    q, k, v = _qkv(gpu, b, tq, tk, h, hkv, hd, dtype, seed=tq)
    spans = _spans(gpu, kind, b, tq, tk)
    for opt in ({}, dict(softcap=5.0), dict(slopes=torch.rand(h, device=gpu) * 0.1)):
        out = attention.attend(q, k, v, spans, scale=0.0, **opt)
        C.check(out, *C.attend(q, k, v, spans, scale=0.0, **opt))


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_scale_of_zero_keeps_what_is_not_a_number(gpu, dtype):
    """0 x inf is NaN: a query that is not finite, and those that see such a key, are NaN; the others do not change."""
    q, k, v = _qkv(gpu, 1, 90, 90, 2, 2, 64, dtype)
    spans = _spans(gpu, "causal", 1, 90, 90)
    ref = attention.attend(q, k, v, spans, scale=0.0)
    q[0, 3, 0, 2], q[0, 4, 0, 7], k[0, 50, 1, 1] = float("inf"), float("nan"), float("-inf")
    out = attention.attend(q, k, v, spans, scale=0.0)
    bad = torch.zeros(90, 2, dtype=torch.bool, device=gpu)
    bad[3:5, 0] = bad[50:, 1] = True
    assert out[0, bad].isnan().all() and torch.equal(out[0, ~bad], ref[0, ~bad])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,n,heads", [(64, 200, 2), (256, 150, 2), (128, 1400, 48)])
def test_a_cap_is_each_scores_own(gpu, dtype, hd, n, heads):
    """Large scores of other queries, or of keys that a query does not see, do not change a bit of its result."""
    q, k, v = _qkv(gpu, 1, n, n, heads, heads, hd, dtype, seed=hd)
    spans = _spans(gpu, "causal", 1, n, n)
    for slopes in (None, torch.rand(heads, device=gpu) * 0.1):
        ref = attention.attend(q, k, v, spans, softcap=50.0, slopes=slopes)
        k2, q2 = k.clone(), q.clone()
        k2[0, n - 10:] *= 300
        assert torch.equal(attention.attend(q, k2, v, spans, softcap=50.0, slopes=slopes)[:, :n - 10], ref[:, :n - 10])
        q2[0, 17] *= 300
        out = attention.attend(q2, k, v, spans, softcap=50.0, slopes=slopes)
        assert torch.equal(out[:, :17], ref[:, :17]) and torch.equal(out[:, 18:], ref[:, 18:])


@pytest.mark.parametrize("softcap", [1.0, 8.0, 100.0])
def test_caps_next_to_the_two_forms_border(gpu, softcap):
    """Scores on both sides of the border in every tile."""
    q, k, v = _qkv(gpu, 1, 150, 150, 2, 2, 128, torch.float16, seed=4)
    for scale in (0.35 * softcap / 128 ** 0.5, 0.05 * softcap):
        for spans in (None, _spans(gpu, "random", 1, 150, 150)):
            C.check(attention.attend(q, k, v, spans, scale=scale, softcap=softcap),
                    *C.attend(q, k, v, spans, scale=scale, softcap=softcap))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tq,tk,heads", [(1, 65536, 2), (500, 65536, 1), (1500, 16384, 48)])
def test_many_keys_of_small_weight_count(gpu, dtype, tq, tk, heads):
    """One key outweighs each of the others by e^18, 2^26: together they are 2^-12 to 2^-10 of the sum, and hold all of its value.

    Rounded: the weights (eps / 2 of the values' type), the result, and, 2^-12 in all, the score of 18 log2(e) (2^-19) and the sums,
    of at most 2^10 terms a lane (2^-14).
    """
    q = torch.ones(1, tq, heads, 64, device=gpu, dtype=dtype)
    k, v = torch.zeros(1, tk, heads, 64, device=gpu, dtype=dtype), torch.ones(1, tk, heads, 64, device=gpu, dtype=dtype)
    k[0, 5], v[0, 5] = 2.25, 0.0  # 64 x 2.25 / 8 = 18
    others = (tk - 1) * math.exp(-18.0)
    want = others / (1 + others)
    out = attention.attend(q, k, v).double()
    assert bool(((out - want).abs() <= want * (torch.finfo(dtype).eps + 2.0 ** -12)).all()), (out.min().item(), out.max().item(), want)
