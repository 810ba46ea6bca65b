"""Attention whose scores are far past 2^22, where neighbouring numbers of fp32 are half a unit and more apart, on the MI355X.

Keys are multiples g_j u of one vector, the best one with g = 1 and the others 10 % or more away, queries are of one sign: the best key's
score leads by a tenth of itself, so that every other weight is 0. The result is then the best key's value itself: its weight relative
to the maximum is 2^0, and what its weight is taken against (a power of two) divides out again.
"""
import pytest
import torch

from flashact_amd import kv8, paged
from tests import kv8_case, paged_case

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
# scores in base 2 with 128 dims, about: 2^23, 2^28.7, 2^30.2, 2^33
SIZES = [(900.0, 700.0), (9000.0, 3000.0), (8000.0, 10000.0), (30000.0, 20000.0)]


def _inputs(gpu, dtype, sizes, tokens, heads, kv_heads, hd, n, best, sign):
    gen = torch.Generator(device=gpu).manual_seed(n + tokens)
    rand = lambda *s: torch.rand(*s, generator=gen, device=gpu)  # noqa: E731
    g = 0.4 + 0.5 * rand(n) if sign > 0 else 1.2 + 0.8 * rand(n)
    g[best] = 1.0
    k = (sizes[1] * g[:, None, None] * (0.5 + rand(kv_heads, hd))).to(dtype)
    v = torch.randn(n, kv_heads, hd, generator=gen, device=gpu).to(dtype)
    q = (sign * sizes[0] * (0.5 + rand(tokens, heads, hd))).to(dtype)
    return q[None], k[None], v[None]


def _lead(q, k, best, scale):
    """The best key leads by more than 5 % of its score in every row."""
    k = k.double().repeat_interleave(q.shape[2] // k.shape[2], 2)
    for h in range(q.shape[2]):
        s = q[0, :, h].double() @ k[0, :, h].t() * scale
        top = s[:, best].clone()
        s[:, best] = -float("inf")
        assert bool((top - s.amax(-1) > 0.05 * top.abs()).all()) and bool((top.abs() > 2.0 ** 21).all())


def _pages(gpu, k, v, width=None):
    n, h, hd = k.shape[1:]
    pool, table = paged_case.filled(gpu, (n,), h, hd, k.dtype, width=width)
    lens = torch.tensor([n], dtype=torch.int32, device=gpu)
    paged.append(pool, table, k, v, torch.zeros_like(lens))
    return pool, table, lens


def _want(v, best, heads, tokens):
    return v[:, best, None].repeat_interleave(heads // v.shape[2], 2).expand(1, tokens, heads, v.shape[3])


# tokens, heads, K/V heads, dims, keys, the table's pages: one row, a tile, tiles, splits joined by the last workgroup and by a kernel, two
# tiles a wave
SHAPES = [(1, 8, 1, 256, 300, None), (3, 6, 2, 128, 700, None), (40, 4, 4, 96, 700, None), (1, 2, 1, 64, 9000, None), (2, 8, 1, 256, 20011, None),
          (40, 8, 1, 128, 700, 4000), (40, 4, 1, 64, 3000, 8192), (45, 3, 1, 96, 300, 8192)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("tokens,heads,kv_heads,hd,n,width", SHAPES)
@pytest.mark.parametrize("sign", [1, -1])
def test_pages(gpu, dtype, sizes, tokens, heads, kv_heads, hd, n, width, sign):
    for best in (3, n // 2):
        q, k, v = _inputs(gpu, dtype, sizes, tokens, heads, kv_heads, hd, n, best, sign)
        _lead(q, k, best, hd ** -0.5)
        pool, table, lens = _pages(gpu, k, v, width)
        assert torch.equal(paged.attend(q, pool, table, lens), _want(v, best, heads, tokens))
        assert torch.equal(paged.attend(-q, pool, table, lens, scale=-1.7), _want(v, best, heads, tokens))
        slopes = torch.full((heads,), 0.5, device=gpu)
        assert torch.equal(paged.attend(q, pool, table, lens, slopes=slopes), _want(v, best, heads, tokens))
        cap = 8.0 * float(q.abs().amax()) * float(k.abs().amax()) * hd ** 0.5
        assert torch.equal(paged.attend(q, pool, table, lens, softcap=cap), _want(v, best, heads, tokens))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("tokens,heads,kv_heads,hd,n,width", SHAPES)
def test_pages_with_two_best_keys(gpu, dtype, sizes, tokens, heads, kv_heads, hd, n, width):
    """Equal keys in two pages have equal scores: half of each value, rounded once."""
    q, k, v = _inputs(gpu, dtype, sizes, tokens, heads, kv_heads, hd, n, 5, 1)
    k[0, n // 2] = k[0, 5]
    pool, table, lens = _pages(gpu, k, v, width)
    half = (0.5 * (v[:, 5:6].float() + v[:, n // 2:n // 2 + 1].float())).to(dtype)
    assert torch.equal(paged.attend(q, pool, table, lens), _want(half, 0, heads, tokens))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,heads,kv_heads,hd,n,width", SHAPES)
def test_large_scores_of_other_rows_change_nothing(gpu, dtype, tokens, heads, kv_heads, hd, n, width):
    """Every other head's queries are small enough for ordinary scores: their results are those of a call without the large ones."""
    q, k, v = _inputs(gpu, dtype, (8000.0, 10000.0), tokens, heads, kv_heads, hd, n, 7, 1)
    pool, table, lens = _pages(gpu, k, v, width)
    q[:, :, ::2] *= 2.0 ** -27 if dtype is torch.bfloat16 else 2.0 ** -24
    alone = q.clone()
    alone[:, :, 1::2] = 0
    both, one = paged.attend(q, pool, table, lens), paged.attend(alone, pool, table, lens)
    assert torch.equal(both[:, :, ::2], one[:, :, ::2])
    kr, vr = paged_case.rows_of(pool, table[:, :(n + 31) // 32])
    kv8_case.check(one, *kv8_case.attend(alone, kr, vr, (n,)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("tokens,heads,kv_heads,hd,n", [(1, 8, 1, 256, 300), (3, 6, 2, 128, 700), (40, 4, 4, 96, 700), (1, 2, 1, 64, 9000)])
def test_codes(gpu, dtype, sizes, tokens, heads, kv_heads, hd, n):
    """The 8-bit cache: codes and scales as they are stored, which 16 bits hold exactly."""
    best = n // 2
    q, k, v = _inputs(gpu, dtype, sizes, tokens, heads, kv_heads, hd, n, best, 1)
    cache = kv8.make_caches(1, 1, n, kv_heads, hd, gpu)[0]
    lens = torch.tensor([n], dtype=torch.int32, device=gpu)
    kv8.store(cache, k, v, torch.zeros_like(lens))
    k, v = (x[:, :n] for x in kv8.load(cache, lens, dtype=torch.float32))
    _lead(q, k, best, hd ** -0.5)
    want = _want(v, best, heads, tokens).to(dtype)
    assert torch.equal(kv8.attend(q, cache, lens), want)
    assert torch.equal(kv8.attend(-q, cache, lens, scale=-1.7), want)
    assert torch.equal(kv8.attend(q, cache, lens, slopes=torch.full((heads,), 0.5, device=gpu)), want)
