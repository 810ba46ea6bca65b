"""``attention.attend`` on the MI355X against attention in 64 bits (tests/span_case.py has the bound)."""
import pytest
import torch

from flashact_amd import _lib, attention
from tests import span_case as C

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _qkv(gpu, b, tq, tk, h, hkv, hd, dtype, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=gpu).to(dtype)  # noqa: E731
    return r(b, tq, h, hd), r(b, tk, hkv, hd), r(b, tk, hkv, hd)


def _random_spans(gpu, b, tq, tk, seed=0):
    """Any spans: empty, reversed, past both ends, single keys."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    a = torch.randint(-5, tk + 5, (b, tq), generator=g, device=gpu)
    n = torch.randint(-3, tk + 8, (b, tq), generator=g, device=gpu)
    n = torch.where(torch.rand(b, tq, generator=g, device=gpu) < 0.2, torch.randint(-1, 2, (b, tq), generator=g, device=gpu), n)
    return torch.stack([a, a + n], -1).to(torch.int32)


def _documents(gpu, lengths, prefix, behind=0):
    t = lambda v: torch.tensor(v, device=gpu)  # noqa: E731
    return attention.prefix_spans(t(lengths), t(prefix), sum(lengths) + behind)


CASES = [
    # b, tq, tk, heads, kv_heads, hd, spans, options
    (1, 1, 1, 1, 1, 64, None, {}),
    (2, 3, 70, 4, 2, 64, None, {}),
    (1, 130, 130, 2, 1, 128, "causal", {}),
    (2, 100, 100, 2, 2, 96, "random", {}),
    (1, 333, 333, 4, 2, 72, "documents", dict(softcap=20.0)),
    (1, 300, 300, 8, 1, 256, "documents", {}),
    (2, 65, 257, 3, 3, 256, "random", dict(slopes=True)),
    (1, 200, 129, 2, 1, 8, "random", {}),
    (3, 77, 401, 6, 2, 104, "random", dict(softcap=5.0, slopes=True)),
    (1, 64, 1000, 2, 2, 40, "causal", dict(slopes=True)),
    (2, 1100, 1100, 32, 4, 64, "documents", {}),      # enough tiles for two blocks of queries a wave
    (1, 1500, 1500, 48, 16, 128, "documents", dict(softcap=50.0)),
    (1, 2100, 2100, 32, 8, 88, "window", dict(scale=0.5)),
    (4, 1030, 515, 16, 4, 128, "random", dict(slopes=True)),
]


def _spans(gpu, kind, b, tq, tk):
    if kind is None:
        return None
    if kind == "random":
        return _random_spans(gpu, b, tq, tk, seed=tq)
    i = torch.arange(tq, device=gpu) + tk - tq
    if kind == "causal":
        return torch.stack([torch.zeros_like(i), i + 1], -1).to(torch.int32)
    if kind == "window":
        return torch.stack([i - 129, i + 1], -1).to(torch.int32)
    return _documents(gpu, [tq // 2 - 9, 1, tq // 3, 0], [tq // 3, 1, 0, 0], tq - (tq // 2 - 8 + tq // 3))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:7]))
def test_attend(gpu, case, dtype):
    b, tq, tk, h, hkv, hd, kind, opt = case
    q, k, v = _qkv(gpu, b, tq, tk, h, hkv, hd, dtype, seed=tq + hd)
    o = dict(opt)
    if o.pop("slopes", False):
        o["slopes"] = torch.rand(h, device=gpu) * 0.1
    spans = _spans(gpu, kind, b, tq, tk)
    out = attention.attend(q, k, v, spans, **o)
    assert out.dtype == dtype and out.shape == q.shape
    C.check(out, *C.attend(q, k, v, spans, **o))
    assert torch.equal(out, attention.attend(q, k, v, spans, **o))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,n,heads", [(64, 200, 2), (128, 300, 2), (256, 150, 2), (128, 1400, 48)])
def test_what_a_query_does_not_see_does_not_reach_it(gpu, dtype, hd, n, heads):
    """Two documents in one tile, one full of infinities and NaN; and causal rows ahead of a bad token."""
    q, k, v = _qkv(gpu, 1, n, n, heads, heads, hd, dtype, seed=hd)
    a = n // 2 + 3
    spans = _documents(gpu, [a, n - a], [a, 0])
    ref = attention.attend(q, k, v, spans)
    k2, v2 = k.clone(), v.clone()
    k2[0, a + 5, 0], k2[0, a + 40, 1, 3] = float("nan"), float("inf")
    v2[0, a + 9, 0, 1], v2[0, a + 20, 1, 2], v2[0, a + 31, 1, 2] = float("nan"), float("inf"), float("-inf")
    out = attention.attend(q, k2, v2, spans)
    assert torch.equal(out[:, :a], ref[:, :a])
    assert torch.equal(out[:, a:a + 5, 0], ref[:, a:a + 5, 0])
    assert out[:, a + 5:, 0].isnan().all()
    # without bad keys: infinities and NaN of values reach exactly the rows that see them, in their dims
    out = attention.attend(q, k, v2, spans)
    C.check(out, *C.attend(q, k, v2, spans))
    assert out[:, a + 9:, 0, 1].isnan().all() and (out[:, a + 20:a + 31, 1, 2] == float("inf")).all()
    assert out[:, a + 31:, 1, 2].isnan().all()


def test_rows_that_see_nothing_are_zero(gpu):
    q, k, v = _qkv(gpu, 2, 150, 60, 2, 1, 96, torch.bfloat16)
    v[:] = float("nan")
    for spans in (torch.zeros(150, 2), torch.full((150, 2), 60.0), torch.tensor([[50.0, 3.0]]).expand(150, 2),
                  torch.tensor([[-9.0, 0.0]]).expand(150, 2)):
        assert not attention.attend(q, k, v, spans.to(gpu, torch.int32)).any()
    assert not attention.attend(q, k[:, :0], v[:, :0]).any()
    assert attention.attend(q[:, :0], k, v).shape == (2, 0, 2, 96)
    assert attention.attend(q[:0], k[:0], v[:0]).shape == (0, 150, 2, 96)


def test_extreme_scores(gpu):
    """Scores of thousands, equal and opposite: the running maximum moves with every tile; masks next to the lowest values."""
    q, k, v = _qkv(gpu, 1, 70, 500, 2, 2, 128, torch.float16, seed=3)
    k = (k * torch.linspace(0, 60, 500, device=gpu)[:, None, None]).half()
    for spans in (None, _random_spans(gpu, 1, 70, 500)):
        C.check(attention.attend(q, k, v, spans, scale=1.0), *C.attend(q, k, v, spans, scale=1.0))
    big = torch.full_like(k, -240.0)
    C.check(attention.attend(big[:, :70], big.neg(), v, None), *C.attend(big[:, :70], big.neg(), v, None))


@pytest.mark.parametrize("softcap", [1e-3, 0.5, 30.0, 1e4, 1e7])
def test_caps_far_from_the_scores(gpu, softcap):
    """Caps that leave nothing of the scores and caps that leave them as they are: a large one must not cost precision."""
    q, k, v = _qkv(gpu, 1, 70, 300, 2, 2, 64, torch.float16, seed=11)
    spans = _random_spans(gpu, 1, 70, 300)
    for scale in (0.125, 4.0):  # within the near form, and past it
        ref, bound = C.attend(q, k, v, spans, scale=scale, softcap=softcap)
        # the tanh is off by 2^-22 of itself near zero and 2^-23 of one else, where it is 0.3 or more: 2^-21 of the score
        plain = C.attend(q, k, v, spans, scale=scale)[1] + 2.0 ** -10 * ref.abs()
        C.check(attention.attend(q, k, v, spans, scale=scale, softcap=softcap), ref, torch.minimum(bound, plain)
                if softcap >= 1e4 else bound)


def test_sizes_of_one_have_no_strides(gpu):
    """A dimension of one element is never stepped, whatever stride its view carries; memory of its own for the output."""
    q, k, v = (torch.randn(1, 5, 2, 64, device=gpu).bfloat16() for _ in range(3))
    odd = [x.as_strided((1, 5, 2, 64), (3, 128, 64, 1)) for x in (q, k, v)]
    assert torch.equal(attention.attend(*odd), attention.attend(q, k, v))
    one = k[:, :1].as_strided((1, 1, 2, 64), (7, 9, 64, 1)), v[:, :1].as_strided((1, 1, 2, 64), (7, 9, 64, 1))
    assert torch.equal(attention.attend(q, *one), attention.attend(q, k[:, :1], v[:, :1]))
    ref = attention.attend(q, k, v)
    assert attention.attend(q, k, v, out=q) is q and torch.equal(q, ref)  # each query is read before it is written
    with pytest.raises(ValueError, match="share memory"):
        attention.attend(q, k, v, out=k)


def test_views_of_one_projection(gpu):
    """Strided views: heads of one projection, samples of a larger batch, every second token, a transposed layout."""
    qkv = torch.randn(2, 90, 10, 128, device=gpu).bfloat16()
    q, k, v = qkv[:, :, :6], qkv[:, :, 6:8], qkv[:, :, 8:]
    ref = attention.attend(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(attention.attend(q, k, v), ref)
    assert torch.equal(attention.attend(q[1:], k[1:], v[1:]), ref[1:])
    every = attention.attend(q[:, ::2], k[:, ::2], v[:, ::2])
    assert torch.equal(every, attention.attend(q[:, ::2].contiguous(), k[:, ::2].contiguous(), v[:, ::2].contiguous()))
    t = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]  # [B][H][T][hd] behind the view
    assert torch.equal(attention.attend(*t), ref)
    one = k[:, :, :1].expand(2, 90, 2, 128)  # a head shared by stride 0
    assert torch.equal(attention.attend(q, one, v), attention.attend(q, one.contiguous(), v.contiguous()))
    out = torch.empty_like(ref)
    assert attention.attend(q, k, v, out=out) is out and torch.equal(out, ref)


def test_prefix_spans(gpu):
    for dev in ("cpu", gpu):
        t = lambda *v: torch.tensor(v, device=dev)  # noqa: E731
        s = attention.prefix_spans(t(3, 0, 4), t(2, 0, 9), 9)
        assert s.dtype == torch.int32
        assert s.tolist() == [[0, 2], [0, 2], [0, 3], [3, 7], [3, 7], [3, 7], [3, 7], [0, 0], [0, 0]]
        assert attention.prefix_spans(t(3, 4), t(0, 4), 5).tolist() == [[0, 1], [0, 2], [0, 3], [3, 5], [3, 5]]  # cut off
        assert attention.prefix_spans(t(5)[:0], t(5)[:0], 2).tolist() == [[0, 0], [0, 0]]



def test_offsets_past_32_bits(gpu):
    """Keys and values in one tensor of more than 2^32 bytes: a token stride of 2^20 elements, 2100 tokens, bytes past 4 GiB."""
    wide = torch.zeros(1, 2100, 1 << 20, dtype=torch.bfloat16, device=gpu)
    k, v = wide[:, :, :128].unflatten(2, (1, 128)), wide[:, :, 128:256].unflatten(2, (1, 128))
    k.copy_(torch.randn(1, 2100, 1, 128, device=gpu))
    v.copy_(torch.randn(1, 2100, 1, 128, device=gpu))
    q = torch.randn(1, 70, 2, 128, device=gpu).bfloat16()
    assert torch.equal(attention.attend(q, k, v), attention.attend(q, k.contiguous(), v.contiguous()))


def test_refuses_on_the_gpu(gpu):
    q, k, v = _qkv(gpu, 2, 8, 8, 4, 2, 64, torch.bfloat16)
    spans = torch.zeros(8, 2, dtype=torch.int32, device=gpu)
    bad = torch.randn(2, 8, 2, 68, device=gpu).bfloat16()[..., :64]
    for kw, err, text in (
            (dict(k=k.half()), TypeError, "like q"), (dict(q=q.float()), TypeError, "q must be"),
            (dict(k=bad), ValueError, "multiples of 8"), (dict(k=k.cpu()), ValueError, "same GPU"),
            (dict(spans=spans.long()), ValueError, "int32"), (dict(spans=spans[:7]), ValueError, "spans"),
            (dict(spans=spans.cpu()), ValueError, "spans"), (dict(slopes=torch.ones(2, device=gpu)), ValueError, "slopes"),
            (dict(out=torch.empty(2, 8, 4, 64, device=gpu)), ValueError, "out must"),
            (dict(softcap=-1.0), ValueError, "softcap"), (dict(scale=-0.1), ValueError, "scale"),
            (dict(scale=float("nan")), ValueError, "scale")):
        with pytest.raises(err, match=text):
            attention.attend(**{"q": q, "k": k, "v": v, **kw})


SPLIT = [
    # few queries over many keys: the keys are split over workgroups
    (1, 1, 5000, 2, 1, 64, None, {}),
    (2, 70, 3001, 4, 2, 128, "random", dict(slopes=True)),
    (1, 64, 9001, 8, 1, 256, "causal", dict(softcap=30.0)),
    (3, 130, 4099, 3, 3, 96, "window", {}),            # spans of few keys: one part each
    (1, 200, 2600, 2, 2, 72, "random", dict(softcap=5.0, slopes=True)),
    (1, 17, 40000, 16, 4, 128, "causal", {}),
    (1, 1100, 2100, 8, 1, 256, "causal", {}),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", SPLIT, ids=lambda c: "-".join(str(x) for x in c[:7]))
def test_few_queries_over_many_keys(gpu, monkeypatch, case, dtype):
    b, tq, tk, h, hkv, hd, kind, opt = case
    assert attention._workspace_bytes(b, tq, tk, h, hd) > 0
    q, k, v = _qkv(gpu, b, tq, tk, h, hkv, hd, dtype, seed=tq + hd)
    o = dict(opt)
    if o.pop("slopes", False):
        o["slopes"] = torch.rand(h, device=gpu) * 0.1
    spans = _spans(gpu, kind, b, tq, tk)
    ref, bound = C.attend(q, k, v, spans, **o)
    out = attention.attend(q, k, v, spans, **o)
    C.check(out, ref, bound)
    assert torch.equal(out, attention.attend(q, k, v, spans, **o))
    monkeypatch.setattr(attention, "_workspace_bytes", lambda *a: 0)  # no workspace, no parts
    C.check(attention.attend(q, k, v, spans, **o), ref, bound)


@pytest.mark.parametrize("hd", [64, 256])
def test_parts_keep_what_is_not_finite(gpu, hd):
    """A stretch of keys that is all NaN, infinities among the values of another, rows that see neither, either or both."""
    tk = 6000
    q, k, v = _qkv(gpu, 1, 40, tk, 2, 2, hd, torch.bfloat16, seed=hd)
    spans = torch.tensor([[0, tk], [0, 2900], [4100, tk], [2900, 4100], [0, 5000], [7, 7]], device=gpu, dtype=torch.int32)
    spans = spans.repeat(7, 1)[:40].contiguous()
    ref = attention.attend(q, k, v, spans)
    k2, v2 = k.clone(), v.clone()
    k2[0, 2900:4100, 0] = float("nan")
    v2[0, 5500, 1, 5], v2[0, 100, 1, 6] = float("inf"), float("-inf")
    out = attention.attend(q, k2, v2, spans)
    row = torch.arange(40, device=gpu) % 6
    bad = (row == 0) | (row == 3) | (row == 4)  # see the NaN keys, of head 0
    assert out[0, bad, 0].isnan().all() and torch.equal(out[0, ~bad, 0], ref[0, ~bad, 0])
    C.check(out[:, :, 1:], *C.attend(q[:, :, 1:], k2[:, :, 1:], v2[:, :, 1:], spans))
    assert (out[0, (row == 0) | (row == 2), 1, 5] == float("inf")).all() and not out[0, row == 5].any()


@pytest.mark.parametrize("tk", [40, 9000])
def test_out_is_q_or_apart_from_it(gpu, tk):
    buf = torch.randn(40 * 4 * 64 + 64, device=gpu).bfloat16()
    q = buf[:40 * 4 * 64].view(1, 40, 4, 64)
    _, k, v = _qkv(gpu, 1, 1, tk, 4, 2, 64, torch.bfloat16)
    ref = attention.attend(q, k, v)
    with pytest.raises(ValueError, match="share memory"):
        attention.attend(q, k, v, out=buf[64:].view(1, 40, 4, 64))
    with pytest.raises(ValueError, match="share memory"):
        attention.attend(q.view(1, 4, 40, 64).transpose(1, 2), k, v, out=q)
    assert attention.attend(q, k, v, out=q) is q and torch.equal(q, ref)


@pytest.mark.parametrize("tq,tk,h,hkv,hd,kind", [(1100, 2100, 8, 1, 256, "causal"), (1000, 4000, 8, 2, 64, "random"),
                                                 (2300, 2300, 8, 1, 256, "documents")])
def test_parts_in_any_workspace(gpu, monkeypatch, tq, tk, h, hkv, hd, kind):
    """The workgroups that share a tile count themselves in memory of any contents: ones, random words, an earlier call's."""
    q, k, v = _qkv(gpu, 1, tq, tk, h, hkv, hd, torch.float16, seed=tk)
    spans = _spans(gpu, kind, 1, tq, tk)
    ref, bound = C.attend(q, k, v, spans)
    need = attention._workspace_bytes(1, tq, tk, h, hd)
    assert need
    ws = torch.full((need,), 255, dtype=torch.uint8, device=gpu)
    real = _lib.run_on

    def run_on(index, fn, a, what):
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
        real(index, fn, a, what)

    monkeypatch.setattr(_lib, "run_on", run_on)
    out = attention.attend(q, k, v, spans)
    C.check(out, ref, bound)
    for i in range(5):
        if i == 2:
            ws.copy_(torch.randint(0, 256, ws.shape, dtype=torch.uint8, device=gpu))
        assert torch.equal(attention.attend(q, k, v, spans), out)


def test_parts_of_inputs_in_turn(gpu):
    """Calls that reuse one another's workspace take no sum of an earlier one."""
    _, k, v = _qkv(gpu, 1, 1, 4096, 8, 1, 128, torch.bfloat16)
    qs = [torch.randn(1, 1024, 8, 128, device=gpu).bfloat16() for _ in range(3)]
    refs = [attention.attend(q, k, v) for q in qs]
    bad = torch.zeros((), dtype=torch.int64, device=gpu)
    for i in range(600):
        j = (i * 7 + i // 5) % 3
        bad += (attention.attend(qs[j], k, v) != refs[j]).any()
    assert not torch.equal(refs[0], refs[1]) and bad.item() == 0
