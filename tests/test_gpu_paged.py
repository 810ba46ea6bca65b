"""The paged cache on the MI355X: rows in (with the rotation) and out, and attention over it, against 64 bits.

The attention is held to the 8-bit cache's bound (``kv8_case.attend``): its weights are rounded to 2^-12 (fp16) or less.
"""
import pytest
import torch

from flashact_amd import paged
from tests import kv8_case
from tests import paged_case as C

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _ints(gpu, *v):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


def _freqs(gpu, dims):
    return paged.frequencies(dims, device=gpu) if dims else None


def _check_append(gpu, pool, table, k, v, start, count, dims, adjacent, q=None):
    freqs = _freqs(gpu, dims)
    whole = [k.shape[1]] * len(start) if count is None else count
    kt, vt, bound = C.append(pool, table, k, v, start, whole, freqs, adjacent)
    out = paged.append(pool, table, k, v, _ints(gpu, *start), None if count is None else _ints(gpu, *count), q=q, freqs=freqs,
                       adjacent=adjacent)
    got_k, got_v = (x.cpu() for x in C.tokens_of(pool))
    C.close(got_k, kt, bound)
    assert torch.equal(got_v.double().nan_to_num(nan=7e9), vt.nan_to_num(nan=7e9))
    if dims == 0:
        assert torch.equal(got_k.double().nan_to_num(nan=7e9), kt.nan_to_num(nan=7e9))
    if q is None:
        assert out is None
        return
    assert out.shape == q.shape and out.is_contiguous() and out.dtype is q.dtype
    for b, s in enumerate(start):
        n = 0 if s < 0 else max(0, min(whole[b], q.shape[1]))
        ref, bound = C.turned(q[b, :n].cpu(), s + torch.arange(n), None if freqs is None else freqs.cpu(), adjacent)
        C.close(out[b, :n].cpu(), ref, bound)
        assert not out[b, n:].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,heads,kv_heads,dims,adjacent", [(256, 8, 1, 256, True), (128, 6, 2, 64, False), (96, 4, 4, 96, False),
                                                             (64, 3, 1, 16, True), (128, 1, 1, 0, False)])
@pytest.mark.parametrize("tokens", [1, 3, 8, 45])
def test_append(gpu, dtype, hd, heads, kv_heads, dims, adjacent, tokens):
    start = (0, 5, 31, 200, 64)
    count = (tokens, max(0, tokens - 1), tokens, tokens + 9, 0)
    pool, table = C.filled(gpu, [s + tokens for s in start], kv_heads, hd, dtype, seed=tokens)
    gen = torch.Generator(device=gpu).manual_seed(hd)
    qkv = torch.randn(len(start), tokens, heads + 2 * kv_heads, hd, generator=gen, device=gpu).to(dtype)
    q, k, v = qkv.split((heads, kv_heads, kv_heads), 2)
    _check_append(gpu, pool, table, k, v, start, count, dims, adjacent, q)
    _check_append(gpu, pool, table, k, v, start, None, dims, adjacent)


@pytest.mark.parametrize("tokens", [1, 40])
def test_append_drops_what_has_no_place(gpu, tokens):
    """Negative starts, rows behind the table's end, pages outside the pool; queries turn all the same, but for negative starts."""
    start = (-1, -2 ** 31, 90, 96, 2 ** 31 - 1, 3, 40)
    pool, table = C.filled(gpu, [96] * len(start), 2, 64, torch.bfloat16, seed=1)
    table[5, 0], table[6, 1] = -7, pool["k"].shape[0]
    before = {n: t.clone() for n, t in pool.items()}
    gen = torch.Generator(device=gpu).manual_seed(5)
    k, v = (torch.randn(len(start), tokens, 2, 64, generator=gen, device=gpu).bfloat16() for _ in range(2))
    q = torch.randn(len(start), tokens, 2, 64, generator=gen, device=gpu).bfloat16()
    _check_append(gpu, pool, table, k, v, start, None, 64, False, q)
    now = {n: t.clone() for n, t in pool.items()}
    if tokens == 1:
        assert sum((now["k"] != before["k"]).any(-1).any(2).any(1).flatten().tolist()) == 1  # sample 2 alone has a place


def test_append_far_positions(gpu):
    """Angles of positions up to 2^23: the queries', whatever the table holds."""
    start = (2 ** 23 - 5, 1000003, 131071, 65535)
    pool, table = C.filled(gpu, [32] * 4, 1, 256, torch.float16, seed=2)
    q = torch.randn(4, 9, 3, 256, device=gpu).half()
    k = torch.randn(4, 9, 1, 256, device=gpu).half()
    _check_append(gpu, pool, table, k, k, start, None, 256, False, q)


def test_append_keeps_what_is_not_finite(gpu):
    pool, table = C.filled(gpu, [40], 1, 64, torch.bfloat16)
    k = torch.randn(1, 40, 1, 64, device=gpu).bfloat16()
    k[0, 3, 0, 5], k[0, 9, 0, 60], k[0, 11, 0, 2] = float("nan"), float("inf"), 3e38
    _check_append(gpu, pool, table, k[..., :], k, (0,), None, 0, False)


def test_append_into_the_last_pages_of_a_large_pool(gpu):
    """Offsets behind 2^31 bytes and elements."""
    pages = (1 << 31) // (32 * 256) + 5
    pool = paged.make_pools(1, pages, 1, 256, device=gpu)[0]
    table = _ints(gpu, pages - 1, pages - 3)[None].contiguous()
    k, v = (torch.randn(1, 50, 1, 256, device=gpu).bfloat16() for _ in range(2))
    paged.append(pool, table, k, v, _ints(gpu, 2))
    for got, want in zip(paged.load(pool, table, _ints(gpu, 52)), (k, v)):
        assert torch.equal(got[:, 2:52], want) and not got[:, 52:].any()
    assert torch.equal(C.tokens_of({n: t[-1:] for n, t in pool.items()})[0][0, 2:, 0], k[0, :30, 0])
    q = torch.randn(1, 1, 4, 256, device=gpu).bfloat16()
    kr, vr = (x[:, 0:50].transpose(1, 2).double() for x in (k, v))
    two = torch.zeros(1, 1, 2, 256, device=gpu, dtype=torch.float64)
    kr, vr = torch.cat([two, kr], 2), torch.cat([two, vr], 2)
    kv8_case.check(paged.attend(q, pool, table, _ints(gpu, 52)), *kv8_case.attend(q, kr, vr, (52,)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,kv_heads", [(256, 1), (96, 3), (64, 2), (128, 2)])
def test_load(gpu, dtype, hd, kv_heads):
    lens = (70, 0, 1, 96, 500, -4)
    pool, table = C.filled(gpu, [96] * len(lens), kv_heads, hd, dtype, seed=hd)
    table[3, 1], table[0, 0] = -1, 1 << 30
    k, v = paged.load(pool, table, _ints(gpu, *lens))
    want = [x.transpose(1, 2) for x in C.rows_of(pool, table)]
    for got, ref in zip((k, v), want):
        assert got.shape == (len(lens), 96, kv_heads, hd)
        for b, n in enumerate(lens):
            n = max(0, min(n, 96))
            assert torch.equal(got[b, :n].double(), ref[b, :n]) and not got[b, n:].any()


def test_load_into_the_denoise_loops_caches(gpu):
    """Views of its layouts, left as they are behind each sample's tokens; rows of any stride."""
    lens = (70, 33, 5)
    pool, table = C.filled(gpu, lens, 1, 256, torch.bfloat16, seed=9, width=4)
    kc = torch.full((3, 2, 80, 256), 7.0, dtype=torch.bfloat16, device=gpu)
    vt = torch.full((3, 2, 256, 80), 7.0, dtype=torch.bfloat16, device=gpu)
    paged.load(pool, table, _ints(gpu, *lens), k=kc[:, 1, :, None], v=vt[:, 1].transpose(1, 2)[:, :, None])
    wide = torch.full((3, 66, 1, 515), 7.0, dtype=torch.bfloat16, device=gpu)
    paged.load(pool, table, _ints(gpu, *lens), k=wide[..., 1:513:2], v=wide[..., 0:512:2])
    k, v = C.rows_of(pool, table)
    for b, n in enumerate(lens):
        assert torch.equal(kc[b, 1, :n].double(), k[b, 0, :n]) and torch.equal(vt[b, 1, :, :n].t().double(), v[b, 0, :n])
        assert (kc[b, 1, n:] == 7).all() and (vt[b, 1, :, n:] == 7).all()
        m = min(n, 66)
        assert torch.equal(wide[b, :m, 0, 1:513:2].double(), k[b, 0, :m]) and (wide[b, m:] == 7).all()
        assert torch.equal(wide[b, :m, 0, 0:512:2].double(), v[b, 0, :m]) and (wide[b, :, :, 513:] == 7).all()
    assert (kc[:, 0] == 7).all() and (vt[:, 0] == 7).all()


def test_load_refuses_what_it_would_overwrite(gpu):
    pool, table = C.filled(gpu, (40,), 1, 64, torch.bfloat16)
    rows = torch.zeros(1, 40, 1, 64, dtype=torch.bfloat16, device=gpu)
    lens = _ints(gpu, 40)
    inside = pool["k"].view(-1)[:40 * 64].view(1, 40, 1, 64)
    for k, v in ((rows, rows), (rows[:, :1].expand(1, 40, 1, 64), rows.clone()), (inside, rows)):
        with pytest.raises(ValueError):
            paged.load(pool, table, lens, k=k, v=v)


# ---------------------------------------------------------------- attention
def _check(gpu, q, pool, table, lens, **kw):
    k, v = C.rows_of(pool, table)
    out = paged.attend(q, pool, table, _ints(gpu, *lens),
                       **{n: (_ints(gpu, *x) if n == "count" and x is not None else x) for n, x in kw.items()})
    kv8_case.check(out, *kv8_case.attend(q, k, v, lens, **kw))
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,heads,kv_heads", [(256, 8, 1), (128, 6, 2), (96, 4, 4), (64, 32, 2)])
@pytest.mark.parametrize("tokens", [1, 3, 50])
@pytest.mark.parametrize("causal", [True, False])
def test_attend(gpu, dtype, hd, heads, kv_heads, tokens, causal):
    lens = (1, 0, 31, 32, 33, 983, 260)
    pool, table = C.filled(gpu, lens, kv_heads, hd, dtype, seed=tokens)
    q = torch.randn(len(lens), tokens, heads, hd, generator=torch.Generator(device=gpu).manual_seed(hd), device=gpu).to(dtype)
    _check(gpu, q, pool, table, lens, causal=causal)
    count = (1, tokens, 0, tokens, -3, tokens + 5, max(1, tokens - 1))
    out = _check(gpu, q, pool, table, lens, causal=causal, count=count, softcap=5.0, slopes=torch.rand(heads, device=gpu) * 0.1)
    for b, n in enumerate(count):
        assert not out[b, max(0, min(n, tokens)):].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,tokens,hd", [((20011,), 1, 256), ((9000, 40), 2, 64), ((3001, 2999, 1), 70, 128)])
def test_attend_long(gpu, dtype, lens, tokens, hd):
    """Keys split over workgroups, joined by the last one or by a kernel; some samples use fewer splits."""
    pool, table = C.filled(gpu, lens, 1, hd, dtype, seed=3)
    q = torch.randn(len(lens), tokens, 4, hd, device=gpu).to(dtype)
    assert paged._workspace_bytes(len(lens), tokens, 4, 1, hd, table.shape[1]) > 0
    _check(gpu, q, pool, table, lens)
    _check(gpu, q, pool, table, lens, scale=0.5, softcap=30.0)
    _check(gpu, q, pool, table, lens, scale=-0.3, slopes=torch.tensor([0.5, -0.01, 0.0, 2.0], device=gpu))


@pytest.mark.parametrize("dtype", DTYPES)
def test_lens_and_tables_of_any_size(gpu, dtype):
    """Lengths behind the table's end count as its end; a wide table, whose rows are a part of wider ones; queries of any stride."""
    pool, table = C.filled(gpu, (100, 64, 30), 2, 64, dtype, width=40)
    q = torch.randn(3, 4, 2, 6, 64, device=gpu).to(dtype)[:, :, 1]
    ref = _check(gpu, q, pool, table, (100, 64, 30))
    wide = torch.full((3, 50), -5, dtype=torch.int32, device=gpu)
    wide[:, 3:43] = table
    assert torch.equal(paged.attend(q, pool, wide[:, 3:43], _ints(gpu, 100, 64, 30)), ref)
    _check(gpu, q, pool, table[:, :2], (64, 64, 30))
    k, v = C.rows_of(pool, table[:, :2])
    out = paged.attend(q, pool, table[:, :2], _ints(gpu, 1000, 2 ** 31 - 1, 30))
    kv8_case.check(out, *kv8_case.attend(q, k, v, (64, 64, 30)))
    assert not paged.attend(q, pool, table, _ints(gpu, -1, -2 ** 31, 0)).any()


def test_shared_pages(gpu):
    """Requests with a common beginning read the same pages; one ends inside a page."""
    pool, table = C.filled(gpu, (320, 40), 1, 128, torch.bfloat16)
    table[1, :6] = table[0, :6]
    q = torch.randn(2, 1, 8, 128, device=gpu).bfloat16()
    _check(gpu, q, pool, table, (320, 170))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 20])
def test_keys_of_no_page_are_not_seen(gpu, dtype, tokens):
    """Holes anywhere: the first page, the last, all of a wave's, all of a sample's. Page 0, read in their place, is full of NaN."""
    pool, table = C.filled(gpu, (700, 700, 33, 700), 1, 64, dtype, seed=4)
    table += 1  # no row names page 0
    for n in ("k", "v"):
        pool[n] = torch.cat([torch.full_like(pool[n][:1], float("nan")), pool[n]])
    table[0, 0], table[0, 5], table[0, 21], table[2, 0], table[1, 3:19] = -1, 1 << 20, -2, -2 ** 31, -1
    table[3] = -1
    q = torch.randn(4, tokens, 4, 64, device=gpu).to(dtype)
    lens = (700, 700, 33, 700)
    out = paged.attend(q, pool, table, _ints(gpu, *lens))
    k, v = C.rows_of(pool, table)
    key = torch.arange(k.shape[2], device=gpu)
    held = ((table >= 0) & (table < pool["k"].shape[0])).repeat_interleave(32, 1)
    for b, n in enumerate(lens):
        pos = n - tokens + torch.arange(tokens, device=gpu)
        ref = C.attend_masked(q[b], k[b], v[b], held[b] & (key <= pos[:, None]))
        # as kv8_case.attend's bound: weights 2^-12, scores of |q| |k| / 8 <= 40 to 2^-17 of it, values below 5
        C.close(out[b], ref, torch.full_like(ref, 5 * (2.0 ** -12 + 3 * 40 * 2.0 ** -17)))
    assert not out[3].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_seen_does_not_reach_a_row(gpu, dtype, what):
    """Keys and values behind a query, and behind the last token in its page, are not finite."""
    lens = (45, 200)
    pool, table = C.filled(gpu, lens, 1, 128, dtype, seed=6)
    kt, vt = C.tokens_of(pool)
    q = torch.randn(2, 5, 4, 128, device=gpu).to(dtype)
    ref = paged.attend(q, pool, table, _ints(gpu, *lens))
    for b, n in enumerate(lens):
        for at in range(n - 2, (n + 31) // 32 * 32):  # the last two tokens: the first three queries do not see them
            page = int(table[b, at // 32])
            pool["v"][page, 0, at % 32 // 8, :, at % 8] = what
            pool["k"][page, 0, :, at % 32] = what
    out = paged.attend(q, pool, table, _ints(gpu, *lens))
    assert torch.equal(out[:, :3], ref[:, :3]) and bool(out[:, 4].isnan().any(-1).all())


@pytest.mark.parametrize("dtype,tokens,length", [(torch.bfloat16, 1, 131072), (torch.float16, 1, 131072), (torch.float16, 40, 20000)])
def test_many_keys_of_small_weight_count(gpu, dtype, tokens, length):
    """One key outweighs each of the others by e^18, 2^26: together they are 2^-11 to 2^-9 of the sum, and hold all of its value."""
    pool = paged.make_pools(1, length // 32, 1, 64, dtype, gpu)[0]
    pool["v"].fill_(1.0)
    pool["k"][0, 0, :, 5], pool["v"][0, 0, 0, :, 5] = 2.25, 0.0  # 64 x 2.25 / 8 = 18
    table = torch.arange(length // 32, device=gpu, dtype=torch.int32)[None]
    q = torch.ones(1, tokens, 8, 64, device=gpu, dtype=dtype)
    out = paged.attend(q, pool, table, _ints(gpu, length), causal=False).double()
    others = (length - 1) * 2.718281828459045 ** -18.0
    want = others / (1 + others)
    # rounded: the weights (2^-12), the result, and, 2^-12 in all, the score (2^-19) and sums of at most 2^10 terms a lane (2^-14)
    assert bool(((out - want).abs() <= want * (torch.finfo(dtype).eps / 2 + 2.0 ** -11)).all()), (out.min().item(), want)


def test_values_next_to_the_ends_of_the_range(gpu):
    pool, table = C.filled(gpu, (3000,), 1, 64, torch.bfloat16, seed=8)
    q = torch.randn(1, 2, 4, 64, device=gpu).bfloat16()
    for factor in (2.0 ** 122, 2.0 ** -95):
        one = {"k": pool["k"], "v": pool["v"] * factor}
        _check(gpu, q, one, table, (3000,))


def test_results_are_the_same_every_time(gpu):
    pool, table = C.filled(gpu, (5000, 100), 1, 256, torch.bfloat16)
    q = torch.randn(2, 1, 8, 256, device=gpu).bfloat16()
    ref = paged.attend(q, pool, table, _ints(gpu, 5000, 100))
    for _ in range(10):
        assert torch.equal(paged.attend(q, pool, table, _ints(gpu, 5000, 100)), ref)
    assert torch.equal(paged.attend(q, pool, table, _ints(gpu, 5000, 100), out=q), ref) and torch.equal(q, ref)


def test_attend_refuses_results_over_what_it_reads(gpu):
    pool, table = C.filled(gpu, (64,), 1, 64, torch.bfloat16)
    q = torch.randn(1, 2, 1, 64, device=gpu).bfloat16()
    lens = _ints(gpu, 64)
    for out in (pool["k"].view(-1)[:128].view(1, 2, 1, 64), pool["v"].view(-1)[64:192].view(1, 2, 1, 64)):
        with pytest.raises(ValueError, match="share"):
            paged.attend(q, pool, table, lens, out=out)
    big = torch.randn(1, 3, 1, 64, device=gpu).bfloat16()
    with pytest.raises(ValueError, match="being it"):
        paged.attend(big[:, :2], pool, table, lens, out=big[:, 1:])
