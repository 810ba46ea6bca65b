"""Outputs that lie over what a call reads, or over each other, are refused; those that lie beside it are not."""
import pytest
import torch

from flashact_amd import attention, kv8, w4

pytestmark = pytest.mark.gpu


def test_a_result_of_another_type_is_not_the_residual(gpu):
    """Shorter elements from the residual's address on: rows would lie over residuals that others still read."""
    x, w = torch.randn(8, 256, device=gpu).bfloat16(), w4.quantize(torch.randn(64, 256, device=gpu))
    res = torch.randn(8, 64, device=gpu)
    ref = w4.linear(x, w, residual=res)
    for t in (torch.bfloat16, torch.float16):
        over = res.view(t).view(-1)[:8 * 64].view(8, 64)
        with pytest.raises(ValueError, match="share memory"):
            w4.linear(x, w, residual=res, out=over)
        assert torch.equal(w4.linear(x, w, residual=res, out=torch.empty(8, 64, dtype=t, device=gpu)), ref.to(t))
    assert w4.linear(x, w, residual=res, out=res) is res and torch.equal(res, ref)


def test_a_product_is_not_written_over_its_bias_or_weights(gpu):
    """The bias is read by every row: the first one that is written would be the others' bias."""
    x, w = torch.randn(3, 256, device=gpu).bfloat16(), w4.quantize(torch.randn(64, 256, device=gpu))
    buf = torch.randn(4 * 64, device=gpu)
    for bias in (buf[:64], buf[128:192]):
        with pytest.raises(ValueError, match="share memory"):
            w4.linear(x, w, bias=bias, out=buf[:192].view(3, 64))
    for part in ("codes", "scales"):
        over = w[part].view(-1).view(torch.bfloat16)[:192].view(3, 64)
        with pytest.raises(ValueError, match="share memory"):
            w4.linear(x, w, out=over)
    bias = buf[192:].clone()
    out = w4.linear(x, w, bias=buf[192:], out=buf[:192].view(3, 64))  # beside it
    assert torch.equal(out, w4.linear(x, w, bias=bias, out_dtype=torch.float32))


def test_attention_is_not_written_over_spans_or_slopes(gpu):
    q, k, v = (torch.randn(1, 40, 2, 64, device=gpu).bfloat16() for _ in range(3))
    out = torch.empty(1, 40, 2, 64, dtype=torch.bfloat16, device=gpu)
    spans, slopes = out.view(-1).view(torch.int32)[:80].view(40, 2), out.view(-1).view(torch.float32)[2000:2002]
    for kw in (dict(spans=spans), dict(slopes=slopes)):
        with pytest.raises(ValueError, match="share memory"):
            attention.attend(q, k, v, out=out, **kw)


def test_attention_is_not_written_over_the_cache_and_its_lengths(gpu):
    cache, lens = kv8.make_caches(1, 2, 64, 2, 64, gpu)[0], torch.tensor([50, 3], dtype=torch.int32, device=gpu)
    q, out = torch.randn(2, 5, 4, 64, device=gpu).bfloat16(), torch.zeros(2, 5, 4, 64, dtype=torch.bfloat16, device=gpu)
    for name in ("k", "v"):
        with pytest.raises(ValueError, match="share memory"):
            kv8.attend(q, cache, lens, out=cache[name].view(-1).view(torch.bfloat16)[:2560].view(2, 5, 4, 64))
    ints = out.view(-1).view(torch.int32)
    for kw in (dict(lens=ints[:2]), dict(count=ints[7:9]), dict(slopes=out.view(-1).view(torch.float32)[20:24]),
               dict(cache=dict(cache, ks=out.view(-1).view(torch.float32)[:8].view(2, 2, 2)))):
        with pytest.raises(ValueError, match="share memory"):
            kv8.attend(**{"q": q, "cache": cache, "lens": lens, "out": out, **kw})


def test_rows_are_not_loaded_over_each_other(gpu):
    """Keys and values that are shifted into one another, and rows that overlap themselves, would be written twice."""
    cache, lens = kv8.make_caches(1, 1, 64, 1, 64, gpu)[0], torch.tensor([60], dtype=torch.int32, device=gpu)
    rows = torch.randn(60, 64, device=gpu)
    kv8.store(cache, rows[None, :, None], rows[None, :, None] * 2, torch.zeros(1, dtype=torch.int32, device=gpu))
    buf = torch.zeros(130, 64, device=gpu)
    part = lambda at: buf[at:at + 60][None, :, None]  # noqa: E731
    with pytest.raises(ValueError, match="no two"):
        kv8.load(cache, lens, k=part(0), v=part(59))
    over = buf.view(-1).as_strided((1, 60, 1, 64), (4096, 32, 64, 1))
    with pytest.raises(ValueError, match="no two"):
        kv8.load(cache, lens, k=over, v=part(70))
    kv8.load(cache, lens, k=part(0), v=part(60))
    k, v = kv8.load(cache, lens, dtype=torch.float32)
    assert torch.equal(buf[:60], k[0, :60, 0]) and torch.equal(buf[60:120], v[0, :60, 0]) and not buf[120:].any()
