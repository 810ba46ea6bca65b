"""paged.attend where each wave has two tiles of 16 rows (pieces of prompts over many pages), against 64 bits.

The choice goes by the table's width, so that short samples in wide tables reach it: 8 or more tiles of a sample and K/V head, and
65536 pages times tiles in all.
"""
import pytest
import torch

from flashact_amd import paged
from tests import kv8_case, paged_case as C
from tests.test_gpu_paged import DTYPES, _check, _ints

pytestmark = pytest.mark.gpu


def _width(samples, tokens, heads, kv_heads):
    tiles = (tokens * (heads // kv_heads) + 15) // 16
    assert tiles >= 8
    return (65536 + tiles * samples * kv_heads - 1) // (tiles * samples * kv_heads)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,heads,kv_heads,tokens", [(128, 8, 1, 17), (128, 6, 2, 50), (96, 4, 4, 130), (64, 32, 2, 8), (64, 12, 1, 13)])
@pytest.mark.parametrize("causal", [True, False])
def test_attend(gpu, dtype, hd, heads, kv_heads, tokens, causal):
    """Pairs of tiles, and one without its second; rows that are not there; samples shorter than their new tokens."""
    lens = (1, 0, 33, 983, 260)
    pool, table = C.filled(gpu, lens, kv_heads, hd, dtype, seed=tokens, width=_width(len(lens), tokens, heads, kv_heads))
    q = torch.randn(len(lens), tokens, heads, hd, generator=torch.Generator(device=gpu).manual_seed(hd), device=gpu).to(dtype)
    full = table
    table = table[:, :31]  # the oracle reads what the table names; behind it there is no page

    def check(**kw):
        k, v = C.rows_of(pool, table)
        out = paged.attend(q, pool, full, _ints(gpu, *lens), **{n: (_ints(gpu, *x) if n == "count" else x) for n, x in kw.items()})
        kv8_case.check(out, *kv8_case.attend(q, k, v, lens, **kw))
        return out

    check(causal=causal)
    count = (1, tokens, tokens - 3, tokens + 5, max(1, tokens // 2))
    out = check(causal=causal, count=count, softcap=5.0, slopes=torch.rand(heads, device=gpu) * 0.1)
    for b, n in enumerate(count):
        assert not out[b, max(0, min(n, tokens)):].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_as_single_tiles(gpu, dtype):
    """A table of its own width (single tiles) and a wide one (pairs) agree to the results' rounding, on several splits."""
    lens = (3001, 700)
    pool, table = C.filled(gpu, lens, 1, 128, dtype, seed=2)
    wide = torch.full((2, 4000), -1, dtype=torch.int32, device=gpu)
    wide[:, :table.shape[1]] = table
    q = torch.randn(2, 30, 8, 128, device=gpu).to(dtype)
    one, two = (paged.attend(q, pool, t, _ints(gpu, *lens)) for t in (table, wide))
    _check(gpu, q, pool, table, lens)
    k, v = C.rows_of(pool, table)
    kv8_case.check(two, *kv8_case.attend(q, k, v, lens))
    for _ in range(5):
        assert torch.equal(paged.attend(q, pool, wide, _ints(gpu, *lens)), two)
    # each is off by half a step of its value, and 2^-12 of the weights on values below 5
    assert bool(((one - two).abs().float() <= torch.finfo(dtype).eps * one.abs().float() + 2 * 5 * 2.0 ** -12).all())
    assert torch.equal(paged.attend(q, pool, wide, _ints(gpu, *lens), out=q), two) and torch.equal(q, two)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_seen_does_not_reach_a_row(gpu, dtype, what):
    """Values behind a query, and behind the last token in its page, are not finite; the rows that see them have what they give."""
    lens, tokens = (45, 200), 20
    pool, table = C.filled(gpu, lens, 1, 128, dtype, seed=6, width=_width(2, tokens, 8, 1))
    q = torch.randn(2, tokens, 8, 128, device=gpu).to(dtype)
    ref = paged.attend(q, pool, table, _ints(gpu, *lens))
    for b, n in enumerate(lens):
        for at in range(n - 5, (n + 31) // 32 * 32):  # the last five tokens: queries up to tokens - 6 do not see them
            page = int(table[b, at // 32])
            pool["v"][page, 0, at % 32 // 8, ::2, at % 8] = what
    out = paged.attend(q, pool, table, _ints(gpu, *lens))
    assert torch.equal(out[:, :tokens - 5], ref[:, :tokens - 5])
    seen = out[:, tokens - 5:]
    assert torch.equal(seen[..., 1::2], ref[:, tokens - 5:, :, 1::2])
    assert bool(seen[..., ::2].isnan().all()) if what != what else bool((seen[..., ::2] == what).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_opposite_infinities_and_holes(gpu, dtype):
    """Two infinities that some rows see both of and others one or none; a page that is none between them."""
    lens, tokens = (160,), 40
    pool, table = C.filled(gpu, lens, 1, 64, dtype, seed=7, width=_width(1, tokens, 4, 1))
    q = torch.randn(1, tokens, 4, 64, device=gpu).to(dtype)
    at = {130: float("inf"), 140: -float("inf")}  # queries are at 120 .. 159
    for n, what in at.items():
        pool["v"][int(table[0, n // 32]), 0, n % 32 // 8, 3, n % 8] = what
    table[0, 2] = -1
    out = paged.attend(q, pool, table, _ints(gpu, *lens))[0, :, :, 3]
    assert bool(torch.isfinite(out[:10]).all()) and bool((out[10:20] == float("inf")).all()) and bool(out[20:].isnan().all())
    k, v = C.rows_of(pool, table[:, :5])
    key, pos = torch.arange(160, device=gpu), 120 + torch.arange(tokens, device=gpu)
    seen = (key <= pos[:, None]) & ((key < 64) | (key >= 96))
    ref = C.attend_masked(q[0], k[0], v[0], seen)
    got = paged.attend(q, pool, table, _ints(gpu, *lens))[0]
    got[..., 3], ref[..., 3] = 0, 0
    # weights 2^-12, scores of |q| |k| / 8 <= 40 to 2^-17 of it, values below 5
    C.close(got, ref, torch.full_like(ref, 5 * (2.0 ** -12 + 3 * 40 * 2.0 ** -17)))
