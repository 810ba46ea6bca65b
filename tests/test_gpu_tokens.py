"""Log probabilities of tokens on the MI355X, against 64 bits (bounds: tokens_case.logprobs)."""
import math

import pytest
import torch

from flashact_amd import tokens
from tests import tokens_case as C

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _logits(gpu, rows, v, dtype, seed=0, stride=None, at=0):
    """N(0, 3^2), rows `stride` apart, from element `at` of the memory on."""
    stride = v if stride is None else stride
    gen = torch.Generator(device=gpu).manual_seed(seed)
    x = (torch.randn(rows * stride + at, generator=gen, device=gpu) * 3).to(dtype)
    return x[at:].view(rows, stride)[:, :v], torch.randint(0, v, (rows,), generator=gen, device=gpu)


def _check(x, t, top, scale=1.0):
    got = tokens.logprobs(x, t, top=top, scale=scale)
    C.check(got, *C.logprobs(x, t, top, scale))
    if not top:
        assert got.top_tokens is None and got.top_logprobs is None
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v,rows", [(1, 3), (2, 1), (7, 5), (255, 2), (4096, 3), (4099, 9), (50021, 2), (262144, 1), (33333, 1100)])
def test_logprobs(gpu, dtype, v, rows):
    x, t = _logits(gpu, rows, v, dtype, seed=v)
    _check(x, t.to(torch.int32), min(v, 8))
    _check(x, t, min(v, 32), 0.7)
    _check(x, t, 0, 1.5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_any_alignment(gpu, dtype):
    for at in range(9):
        x, t = _logits(gpu, 5, 1003, dtype, seed=at, stride=1003 + at, at=at)
        _check(x, t, 5)
    x, t = _logits(gpu, 2, 40001, dtype, stride=40007, at=3)
    _check(x, t, 20)
    x, t = _logits(gpu, 6, 513, dtype)
    got = tokens.logprobs(x.contiguous().view(2, 3, 513), t.view(2, 3), top=4)
    ref = tokens.logprobs(x, t, top=4)
    assert got.logprob.shape == (2, 3) and got.top_tokens.shape == (2, 3, 4)
    for a, b in zip(got, ref):
        assert torch.equal(a.view(b.shape), b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [700, 100003])
def test_ties_go_to_the_lowest_index(gpu, dtype, v):
    """Few different values, all equal ones, sorted rows in both directions."""
    gen = torch.Generator(device=gpu).manual_seed(v)
    few = torch.randint(-2, 3, (3, v), generator=gen, device=gpu).to(dtype)
    same = torch.full((1, v), 1.5, device=gpu, dtype=dtype)
    up = (torch.arange(v, device=gpu) / v * 20).to(dtype)[None]
    zero = torch.where(torch.rand(1, v, generator=gen, device=gpu) < 0.5, 0.0, -0.0).to(dtype)
    x = torch.cat([few, same, up, up.flip(1), zero])
    t = torch.randint(0, v, (x.shape[0],), generator=gen, device=gpu)
    for k in (1, 17, 32):
        _check(x, t, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [40, 9001, 100003])
def test_tokens_that_are_ruled_out(gpu, dtype, v):
    """All but a few, all but one, all of a row; the tokens asked for among them."""
    x, t = _logits(gpu, 6, v, dtype, seed=v)
    x[0, torch.rand(v, device=gpu) < 0.9] = -math.inf
    x[1, 3:] = -math.inf
    x[2, :v - 1] = -math.inf
    x[3] = -math.inf
    x[4, :] = torch.finfo(dtype).min
    x[5, 1:] = torch.finfo(dtype).min
    t[:3] = torch.tensor([0, 2, v - 1])
    got = _check(x, t, 20)
    assert got.logprob[3] == -math.inf and got.entropy[3] == 0 and got.top_tokens[3].tolist() == list(range(20))
    assert got.entropy[2] == 0 and got.logprob[2] == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [60, 70001])
def test_tokens_that_are_none_and_logits_that_are_no_number(gpu, dtype, v):
    x, _ = _logits(gpu, 6, v, dtype, seed=1)
    t = torch.tensor([-1, v, 2 ** 40, -2 ** 40, 0, v - 1], device=gpu)
    got = _check(x, t, 3)
    assert got.logprob[:4].tolist() == [-math.inf] * 4
    ref = tokens.logprobs(x, t, top=12)
    y = x.clone()
    y[1, 5], y[2, v - 1], y[3] = math.nan, math.inf, math.nan
    y[3, 7] = 1.0
    got = tokens.logprobs(y, t.clamp(0, v - 1), top=12)
    for r in (1, 2, 3):
        assert math.isnan(got.logprob[r]) and math.isnan(got.entropy[r]) and bool(got.top_logprobs[r, :1].isnan().all())
    assert got.top_tokens[3].tolist() == [7] + [-1] * 11
    assert got.top_tokens[2, 0] == v - 1
    best = torch.sort(x[1].double().index_fill(0, torch.tensor([5], device=gpu), -math.inf), descending=True, stable=True)[1][:12]
    assert torch.equal(got.top_tokens[1].long(), best)
    for r in (0, 4, 5):
        assert torch.equal(got.top_tokens[r], ref.top_tokens[r]) and torch.equal(got.top_logprobs[r], ref.top_logprobs[r])


@pytest.mark.parametrize("dtype", DTYPES)
def test_logits_of_any_size(gpu, dtype):
    """Far from zero, far apart, and nearly equal; temperatures at both ends."""
    x, t = _logits(gpu, 5, 3001, dtype, seed=5)
    big = 200.0 if dtype is torch.bfloat16 else 30000.0
    y = torch.stack([x[0] + big, x[1] - big, x[2] * 1000, x[3] * 1e-3, x[4]]).to(dtype)
    for scale in (1.0, 1e-4, 50.0):
        _check(y, t, 10, scale)


def test_nothing_and_the_same_every_time(gpu):
    x, t = _logits(gpu, 3, 100003, torch.bfloat16)
    ref = tokens.logprobs(x, t, top=20)
    for _ in range(20):
        for a, b in zip(tokens.logprobs(x, t, top=20), ref):
            assert torch.equal(a, b)
    got = tokens.logprobs(x[:0], t[:0], top=4)
    assert got.logprob.shape == (0,) and got.top_tokens.shape == (0, 4)
    same = tokens.logprobs(x[:1].expand(3, 100003), t, top=3)
    assert torch.equal(same.entropy[0], same.entropy[2])


def test_offsets_behind_32_bits(gpu):
    """Rows that lie 2^31 elements apart."""
    x = torch.zeros((1 << 31) + 1000, dtype=torch.float16, device=gpu)
    rows = torch.as_strided(x, (2, 1000), (1 << 31, 1))
    rows.copy_(torch.randn(2, 1000, device=gpu))
    _check(rows, torch.tensor([5, 999], device=gpu), 7)
