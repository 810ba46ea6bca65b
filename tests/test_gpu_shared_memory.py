"""Outputs that lie over what a call reads, or over each other, are refused; those that lie beside it are not."""
import pytest
import torch

from flashact_amd import w4

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
