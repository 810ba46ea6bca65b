"""The 8-bit cache on the MI355X: ``kv8.store`` and ``kv8.load`` bit for bit against their definition in plain torch,
``kv8.attend`` against attention in 64 bits over the values that the codes stand for (bounds: tests/kv8_case.py)."""
import pytest
import torch

from flashact_amd import _lib, kv8, pi05
from tests import kv8_case as C

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _ints(gpu, *v):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


def _filled(gpu, batch, tokens, heads=1, hd=256, seed=0, spread=1.0):
    """A cache of random codes (NaN codes only where asked for) and random powers of two."""
    g = torch.Generator().manual_seed(seed)
    c = kv8.make_caches(1, batch, tokens, heads, hd, gpu)[0]
    for k in ("k", "v"):
        x = (torch.randn(c[k].shape, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        c[k].copy_(x)
    for k in ("ks", "vs"):
        c[k].copy_(2.0 ** torch.randint(-8, -5, c[k].shape, generator=g).float() * spread)
    return c


def _store_both(gpu, cache, k, v, start, count=None):
    """Stores on the GPU and by the rule; codes, scales and tokens behind must be equal."""
    kc, vc = C.rows_of(cache)
    ks, vs = cache["ks"].cpu().clone(), cache["vs"].cpu().clone()
    n = [k.shape[1]] * k.shape[0] if count is None else count
    C.store(kc, ks, k, start, n)
    C.store(vc, vs, v, start, n)
    kv8.store(cache, k, v, _ints(gpu, *start), None if count is None else _ints(gpu, *count))
    gk, gv = C.rows_of(cache)
    for got, want, name in ((gk, kc, "k"), (gv, vc, "v")):
        # NaN has two codes, which stand for the same
        same = (got == want) | (((got & 127) == 127) & ((want & 127) == 127))
        assert bool(same.all()), (name, same.logical_not().nonzero()[:4].tolist())
    assert torch.equal(cache["ks"].cpu(), ks) and torch.equal(cache["vs"].cpu(), vs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,hd", [(1, 256), (2, 64), (3, 96), (4, 128)])
def test_store_matches_its_definition(gpu, dtype, heads, hd):
    g = torch.Generator(device=gpu).manual_seed(hd)
    rand = lambda *s: torch.randn(*s, generator=g, device=gpu)  # noqa: E731
    for tokens, start in ((1, (0, 5, 31)), (33, (0, 31, 17)), (7, (30, 64, 96)), (64, (0, 1, 40))):
        cache = _filled(gpu, 3, 128, heads, hd, seed=tokens)
        grow = 2.0 ** torch.randint(-6, 6, (3, tokens, 1, 1), generator=g, device=gpu).float()
        _store_both(gpu, cache, (rand(3, tokens, heads, hd) * grow).to(dtype), (rand(3, tokens, heads, hd) / grow).to(dtype), start)


def test_store_token_by_token(gpu):
    """Forty tokens one at a time: growing scales recode the block's earlier ones again and again."""
    cache = kv8.make_caches(1, 2, 64, 1, 128, gpu)[0]
    g = torch.Generator(device=gpu).manual_seed(7)
    for i in range(40):
        k, v = (torch.randn(2, 1, 1, 128, generator=g, device=gpu).mul(1.3 ** i).bfloat16() for _ in range(2))
        _store_both(gpu, cache, k, v, (i, i + 3))


def test_store_counts_ends_and_strides(gpu):
    g = torch.Generator(device=gpu).manual_seed(8)
    qkv = torch.randn(4, 50, 9, 96, generator=g, device=gpu).bfloat16()
    k, v = qkv[:, :, 5:7], qkv[:, :, 7:9]  # views of one projection
    # fewer rows than given; none; rows past the cache's end; a negative start; a start behind the end
    _store_both(gpu, _filled(gpu, 4, 96, 2, 96), k, v, (3, 10, 70, 60), (40, 0, 50, 50))
    _store_both(gpu, _filled(gpu, 4, 96, 2, 96), k, v, (-1, 96, 2000000000, 95), (50, 50, 50, -7))
    # 2-byte aligned rows, and values as the denoise loop's transposed cache holds them
    odd = torch.randn(4, 50, 2, 97, generator=g, device=gpu).bfloat16()[..., 1:]
    vt = torch.randn(4, 2, 96, 64, generator=g, device=gpu).bfloat16().permute(0, 3, 1, 2)[:, :50]
    _store_both(gpu, _filled(gpu, 4, 96, 2, 96), odd, vt, (0, 1, 33, 40))
    _store_both(gpu, _filled(gpu, 4, 96, 2, 96), k[:, :0], v[:, :0], (0, 1, 2, 3))


def test_store_of_what_is_not_finite_and_of_extremes(gpu):
    k = torch.randn(1, 40, 1, 64, device=gpu)
    k[0, 3, 0, 5], k[0, 3, 0, 6], k[0, 35, 0, 1] = float("inf"), float("nan"), float("-inf")
    v = torch.zeros(1, 40, 1, 64, device=gpu)  # a block of zeros
    _store_both(gpu, kv8.make_caches(1, 1, 64, 1, 64, gpu)[0], k, v, (0,))
    huge, tiny = torch.full_like(k, 3.4e38), torch.full_like(k, 1e-38)
    _store_both(gpu, kv8.make_caches(1, 1, 64, 1, 64, gpu)[0], huge, tiny, (0,))
    # 448 * 2^e is the last value of a scale, the next fp32 value needs the next
    edge = torch.full((1, 64, 1, 64), 448.0 * 2.0 ** -3, device=gpu)
    edge[0, 32:] = torch.nextafter(edge[0, 32:], torch.full_like(edge[0, 32:], 1e9))
    _store_both(gpu, kv8.make_caches(1, 1, 64, 1, 64, gpu)[0], edge, -edge, (0,))


@pytest.mark.parametrize("dtype", DTYPES)
def test_load(gpu, dtype):
    for heads, hd in ((1, 256), (2, 64), (3, 96), (4, 128)):
        cache = _filled(gpu, 3, 100, heads, hd, seed=hd)
        codes = C.rows_of(cache)
        lens = (100, 37, 0)
        want = [C.values(c, s).permute(0, 2, 1, 3).float().to(dtype) for c, s in zip(codes, (cache["ks"], cache["vs"]))]
        got = kv8.load(cache, _ints(gpu, *lens), dtype=dtype)
        for x, y in zip(got, want):
            assert x.dtype == dtype and x.shape == (3, 128, heads, hd)
            for b, n in enumerate(lens):
                assert torch.equal(x[b, :n].cpu(), y[b, :n]) and not x[b, n:].any()
        # into rows that are there, of odd alignment: what lies behind lens stays
        k, v = (torch.full((3, 70, heads, hd + 1), 7.0, dtype=dtype, device=gpu) for _ in range(2))
        kv8.load(cache, _ints(gpu, 200, 37, -5), k=k[..., 1:], v=v[..., 1:])
        for x, y in ((k, want[0]), (v, want[1])):
            assert (x[..., 0] == 7).all()
            for b, n in enumerate((70, 37, 0)):
                assert torch.equal(x[b, :n, :, 1:].cpu(), y[b, :n]) and (x[b, n:] == 7).all()


def test_round_trip_with_the_denoise_caches(gpu):
    """bf16 caches of the denoise loop (values transposed) into the 8-bit cache and back."""
    kv = torch.randn(1, 2, 77, 256, device=gpu).bfloat16()
    kc, vt = pi05.make_caches(kv, 80)
    cache = kv8.make_caches(1, 1, 80, device=gpu)[0]
    kv8.store(cache, kc[:, :77, None], vt.transpose(1, 2)[:, :77, None], _ints(gpu, 0))
    k2, v2 = torch.zeros_like(kc), torch.zeros_like(vt)
    kv8.load(cache, _ints(gpu, 77), k=k2[:, :, None], v=v2.transpose(1, 2)[:, :, None])
    for x, y in ((kc[0, :77], k2[0, :77]), (vt[0, :, :77], v2[0, :, :77])):
        # half a step of 2^-3 where normal, half the smallest step at the block's scale (max / 448 < s <= max / 224) below
        assert bool(((x - y).float().abs() <= 2.0 ** -4 * x.float().abs() + 2.0 ** -10 * x.float().abs().max() / 224).all())
    assert not k2[0, 77:].any() and not v2[0, :, 77:].any()


CASES = [
    # batch, tokens, heads, kv_heads, hd, lens, options
    (1, 1, 8, 1, 256, (983,), {}),
    (3, 1, 8, 1, 256, (1, 33, 64), {}),
    (4, 1, 4, 4, 64, (0, 1, 500, 32), dict(slopes=True)),
    (2, 1, 6, 2, 96, (31, 1500), dict(softcap=5.0)),
    (3, 3, 6, 2, 96, (2, 300, 65), dict(slopes=True, softcap=20.0)),
    (2, 7, 16, 4, 128, (7, 999), {}),
    (2, 50, 8, 1, 256, (1018, 301), dict(causal=False)),
    (2, 20, 8, 1, 256, (1018, 11), {}),
    (2, 5, 40, 2, 64, (64, 97), dict(causal=False, slopes=True)),
    (1, 1, 64, 1, 128, (4097,), dict(scale=0.3, softcap=30.0)),
    (2, 1, 2, 2, 256, (20000, 5), {}),
    (3, 6, 2, 1, 128, (100, 4, 60), dict(count=(2, 6, 0))),
    (3, 6, 2, 1, 128, (100, 4, 60), dict(count=(3, 9, -1), causal=False, slopes=True)),
]


def _options(gpu, heads, opt):
    o = dict(opt)
    if o.pop("slopes", False):
        o["slopes"] = torch.rand(heads, device=gpu) * 0.1
    if "count" in o:
        o["count"] = _ints(gpu, *o["count"])
    return o


@pytest.mark.parametrize("dtype", DTYPES[:2])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:5]))
def test_attend(gpu, case, dtype):
    batch, tokens, heads, kv_heads, hd, lens, opt = case
    cache = _filled(gpu, batch, max(max(lens), 1), kv_heads, hd, seed=heads)
    q = torch.randn(batch, tokens, heads, hd, device=gpu).to(dtype)
    o = _options(gpu, heads, opt)
    out = kv8.attend(q, cache, _ints(gpu, *lens), **o)
    kc, vc = C.rows_of(cache)
    ref, bound = C.attend(q, C.values(kc, cache["ks"]).to(gpu), C.values(vc, cache["vs"]).to(gpu), lens, **o)
    C.check(out, ref, bound)
    assert torch.equal(out, kv8.attend(q, cache, _ints(gpu, *lens), **o))


@pytest.mark.parametrize("causal", [True, False])
def test_attend_next_to_what_must_not_be_read(gpu, causal):
    """NaN codes and wild scales behind the last token, NaN in a token that later queries alone see."""
    cache = _filled(gpu, 2, 256, 2, 128, seed=3)
    lens, q = (70, 129), torch.randn(2, 9, 4, 128, device=gpu).bfloat16()
    kc, vc = (x.clone() for x in C.rows_of(cache))
    for b, n in enumerate(lens):
        kc[b, :, n:], vc[b, :, n:] = 0x7F, 0xFF
        vc[b, 1, n - 3, 5] = 0x7F  # a NaN that is held: seen by the last three queries, or by all
        kc[b, 0, n - 2, 7] = 0x7F  # scores of the last two queries of the first head
        cache["ks"][b, :, (n + 31) // 32:] = float("nan")
        cache["vs"][b, :, (n + 31) // 32:] = float("inf")
    cache["k"].copy_(kc.view(2, 2, 8, 32, 8, 16).transpose(3, 4))
    cache["v"].copy_(vc.view(2, 2, 8, 32, 128).transpose(3, 4))
    out = kv8.attend(q, cache, _ints(gpu, *lens), causal=causal)
    ks, vs = cache["ks"].clone(), cache["vs"].clone()
    ks[~torch.isfinite(ks)], vs[~torch.isfinite(vs)] = 1.0, 1.0
    ref, bound = C.attend(q, C.values(kc, ks).to(gpu), C.values(vc, vs).to(gpu), lens, causal=causal)
    C.check(out, ref, bound)
    seen = 3 if causal else 9
    assert out[:, 9 - seen:, 2:, 5].isnan().all() and out[:, :9 - seen, 2:].isfinite().all()


def test_attend_over_scales_that_differ_widely(gpu):
    """Blocks whose scales differ by 2^60, in keys and values: fp16 weights times codes must not lose the small ones."""
    cache = _filled(gpu, 1, 96, 1, 64, seed=5)
    cache["ks"].copy_(torch.tensor([[[2.0 ** -40, 2.0 ** -9, 2.0 ** -50]]]))
    cache["vs"].copy_(torch.tensor([[[2.0 ** 30, 2.0 ** -30, 1.0]]]))
    kc, vc = C.rows_of(cache)
    for q in (torch.randn(1, 1, 4, 64, device=gpu).bfloat16(), 30 * torch.randn(1, 1, 4, 64, device=gpu).bfloat16()):
        out = kv8.attend(q, cache, _ints(gpu, 96))
        ref, bound = C.attend(q, C.values(kc, cache["ks"]).to(gpu), C.values(vc, cache["vs"]).to(gpu), (96,))
        C.check(out, ref, bound)



def test_attend_views(gpu):
    cache = _filled(gpu, 2, 600, 2, 128, seed=6)
    qkv = torch.randn(2, 3, 12, 128, device=gpu).bfloat16()
    q, lens = qkv[:, :, 2:10], _ints(gpu, 600, 217)
    ref = kv8.attend(q.contiguous(), cache, lens)
    assert torch.equal(kv8.attend(q, cache, lens), ref)
    out = torch.empty_like(ref)
    assert kv8.attend(q, cache, lens, out=out) is out and torch.equal(out, ref)


@pytest.mark.parametrize("softcap", [1e-3, 30.0, 1e7])
def test_attend_caps_far_from_the_scores(gpu, softcap):
    cache = _filled(gpu, 1, 200, 1, 64, seed=12)
    q = torch.randn(1, 2, 4, 64, device=gpu).half()
    kc, vc = C.rows_of(cache)
    k, v = C.values(kc, cache["ks"]).to(gpu), C.values(vc, cache["vs"]).to(gpu)
    for scale in (0.05, 2.0, -0.3):
        ref, bound = C.attend(q, k, v, (200,), scale=scale, softcap=softcap)
        plain = C.attend(q, k, v, (200,), scale=scale)[1] + 2.0 ** -10 * ref.abs()  # the tanh is off by 2^-21 of the score
        out = kv8.attend(q, cache, _ints(gpu, 200), scale=scale, softcap=softcap)
        C.check(out, ref, torch.minimum(bound, plain) if softcap >= 1e4 else bound)


def test_sizes_of_one_and_shared_memory(gpu):
    cache = _filled(gpu, 1, 64, 1, 128, seed=13)
    q = torch.randn(1, 1, 4, 128, device=gpu).bfloat16()
    lens = _ints(gpu, 50)
    ref = kv8.attend(q, cache, lens)
    assert torch.equal(kv8.attend(q.as_strided((1, 1, 4, 128), (3, 5, 128, 1)), cache, lens), ref)
    assert kv8.attend(q, cache, lens, out=q) is q and torch.equal(q, ref)  # each query is read before it is written
    rows = torch.zeros(1, 1, 1, 128, device=gpu).expand(1, 64, 1, 128)
    with pytest.raises(ValueError, match="may be one"):
        kv8.load(cache, lens, k=rows, v=rows)


def test_long_cache_past_32_bit_offsets(gpu):
    """A cache of more than 4 GiB of codes: 9 samples of 2^20 + 64 tokens."""
    tokens = (1 << 20) + 64
    cache = kv8.make_caches(1, 9, tokens, 1, 256, gpu)[0]
    for n in ("k", "v"):
        cache[n].copy_(torch.randint(0, 0x70, (1, 1, 1, *cache[n].shape[3:]), device=gpu, dtype=torch.uint8))
    cache["ks"].fill_(2.0 ** -8)
    cache["vs"].fill_(2.0 ** -8)
    at = tokens - 20
    k, v = (torch.randn(9, 2, 1, 256, device=gpu).bfloat16() for _ in range(2))
    start = _ints(gpu, *([at] * 8 + [at - 1]))
    kv8.store(cache, k, v, start)
    tail = {n: cache[n][8:, :, -2:].contiguous() for n in cache}
    kc, vc = C.rows_of(tail)
    ref = C.values(kc, tail["ks"])[0, 0, 64 - 21:64 - 19], C.values(vc, tail["vs"])[0, 0, 64 - 21:64 - 19]
    for got, x in zip(ref, (k, v)):
        assert bool(((got - x[8, :, 0].cpu().double()).abs() <= 2.0 ** -4 * x[8, :, 0].cpu().double().abs() + 2.0 ** -9).all())
    # a key far behind 4 GiB that outweighs all others decides the result
    q = torch.zeros(9, 1, 1, 256, device=gpu, dtype=torch.bfloat16)
    q[8] = k[8, 1, 0] * 20
    out = kv8.attend(q, cache, start + 2, scale=1.0)
    want = ref[1][1].to(gpu)  # the second of the two new tokens
    assert bool(((out[8, 0, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -9).all())


def test_refusals_on_the_gpu(gpu):
    cache = kv8.make_caches(1, 2, 64, 2, 128, gpu)[0]
    k = torch.randn(2, 3, 2, 128, device=gpu).bfloat16()
    at = _ints(gpu, 0, 0)
    for kw, err, text in ((dict(k=k.cpu()), ValueError, "GPU"), (dict(start=at.cpu()), ValueError, "GPU"),
                          (dict(start=at.long()), ValueError, "int32"), (dict(count=at[:1]), ValueError, "int32"),
                          (dict(v=k.float()), TypeError, "both be"), (dict(v=k[:, :2]), ValueError, "must be")):
        with pytest.raises(err, match=text):
            kv8.store(cache, **{"k": k, "v": k, "start": at, **kw})
    q = torch.randn(2, 1, 4, 128, device=gpu).bfloat16()
    for kw, err, text in ((dict(q=q.float()), TypeError, "q must be"), (dict(q=q[:, :, :3]), ValueError, "multiple of 2"),
                          (dict(q=torch.randn(2, 1, 4, 256, device=gpu).bfloat16()[..., ::2]), ValueError, "contiguous"),
                          (dict(q=torch.randn(2, 1, 4, 132, device=gpu).bfloat16()[..., :128]), ValueError, "multiples of 8"),
                          (dict(softcap=-1.0), ValueError, "softcap"), (dict(softcap=float("nan")), ValueError, "softcap"),
                          (dict(slopes=torch.ones(3, device=gpu)), ValueError, "slopes"),
                          (dict(out=torch.empty(2, 1, 4, 128, device=gpu)), ValueError, "out must be"),
                          (dict(lens=at.cpu()), ValueError, "GPU")):
        with pytest.raises(err, match=text):
            kv8.attend(**{"q": q, "cache": cache, "lens": at, **kw})
    assert kv8.attend(q[:, :0], cache, at).shape == (2, 0, 4, 128)


@pytest.mark.parametrize("b,tokens,h,hkv,hd,length", [(1, 200, 8, 1, 64, 1100), (3, 45, 16, 1, 96, 333), (1, 33, 6, 3, 128, 90),
                                                      (2, 70, 32, 4, 64, 5000)])
def test_attend_many_rows(gpu, b, tokens, h, hkv, hd, length):
    """Many row tiles of few samples and heads, which are dealt to the XCDs in runs: the last run is not full."""
    cache = _filled(gpu, b, length, hkv, hd, seed=tokens)
    q = torch.randn(b, tokens, h, hd, generator=torch.Generator(device=gpu).manual_seed(1), device=gpu).bfloat16()
    lens = [length - 7 * i for i in range(b)]
    kc, vc = C.rows_of(cache)
    k, v = C.values(kc, cache["ks"]).to(gpu), C.values(vc, cache["vs"]).to(gpu)
    for causal in (True, False):
        out = kv8.attend(q, cache, _ints(gpu, *lens), causal=causal)
        C.check(out, *C.attend(q, k, v, lens, causal=causal))


def test_shared_memory_is_refused_but_for_q_itself(gpu):
    cache = _filled(gpu, 1, 500, 2, 64, seed=9)
    lens = _ints(gpu, 500)
    buf = torch.randn(4 * 8 * 64 + 64, device=gpu).bfloat16()
    q = buf[:4 * 8 * 64].view(1, 4, 8, 64)
    ref = kv8.attend(q, cache, lens)
    with pytest.raises(ValueError, match="share memory"):
        kv8.attend(q, cache, lens, out=buf[64:].view(1, 4, 8, 64))
    with pytest.raises(ValueError, match="share memory"):
        kv8.attend(q.view(1, 8, 4, 64).transpose(1, 2), cache, lens, out=q)
    assert kv8.attend(q, cache, lens, out=q) is q and torch.equal(q, ref)
    k = torch.empty(1, 500, 2, 64, device=gpu)
    with pytest.raises(ValueError, match="no two"):
        kv8.load(cache, lens, k=k, v=k)
    both = torch.empty(1, 500, 2, 2, 64, device=gpu)  # interleaved: different elements
    kv8.load(cache, lens, k=both[:, :, 0], v=both[:, :, 1])
    want = kv8.load(cache, lens, dtype=torch.float32)
    assert torch.equal(both[:, :, 0], want[0][:, :500]) and torch.equal(both[:, :, 1], want[1][:, :500])


@pytest.mark.parametrize("b,tokens,h,hkv,hd,length", [(1, 1, 8, 1, 256, 983), (4, 50, 8, 1, 256, 900), (5, 1, 16, 4, 128, 1500)])
def test_split_sums_in_any_workspace(gpu, monkeypatch, b, tokens, h, hkv, hd, length):
    """The workgroups that share a row tile count themselves in memory of any contents: ones, random words, an earlier call's."""
    cache = _filled(gpu, b, length, hkv, hd, seed=hd)
    q, lens = torch.randn(b, tokens, h, hd, device=gpu).half(), _ints(gpu, *[length - 200 * i for i in range(b)])
    kc, vc = C.rows_of(cache)
    ref, bound = C.attend(q, C.values(kc, cache["ks"]).to(gpu), C.values(vc, cache["vs"]).to(gpu), lens.tolist())
    need = kv8._workspace_bytes(b, tokens, h, hkv, hd, cache["v"].shape[2])
    assert need
    ws = torch.full((need,), 255, dtype=torch.uint8, device=gpu)
    real = _lib.run_on

    def run_on(index, fn, a, what):
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
        real(index, fn, a, what)

    monkeypatch.setattr(_lib, "run_on", run_on)
    out = kv8.attend(q, cache, lens)
    C.check(out, ref, bound)
    for i in range(5):
        if i == 2:
            ws.copy_(torch.randint(0, 256, ws.shape, dtype=torch.uint8, device=gpu))
        assert torch.equal(kv8.attend(q, cache, lens), out)


def test_split_sums_of_inputs_in_turn(gpu):
    """Calls that reuse one another's workspace take no sum of an earlier one."""
    cache, lens = _filled(gpu, 3, 1000, 1, 256, seed=2), _ints(gpu, 1000, 777, 40)
    qs = [torch.randn(3, 5, 8, 256, device=gpu).bfloat16() for _ in range(3)]
    refs = [kv8.attend(q, cache, lens) for q in qs]
    bad = torch.zeros((), dtype=torch.int64, device=gpu)
    for i in range(600):
        j = (i * 7 + i // 5) % 3
        bad += (kv8.attend(qs[j], cache, lens) != refs[j]).any()
    assert not torch.equal(refs[0], refs[1]) and bad.item() == 0
