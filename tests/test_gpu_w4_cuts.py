"""``w4.linear`` on both sides of the sizes where its products are cut differently (the bound: tests/test_gpu_w4.py)."""
import pytest
import torch

from flashact_amd import w4
from tests.test_gpu_w4 import _check, _reference

pytestmark = pytest.mark.gpu

SIZES = [
    # rows of weights, columns: tiles of 16 and chunks of 128
    (496, 14336), (512, 14336), (512, 14208), (3200, 16384), (3216, 16384), (3216, 20480), (4096, 16384), (4112, 16384), (16368, 264),
    (16384, 264), (32752, 1024), (32768, 1024), (32768, 1032),
]


@pytest.mark.parametrize("n,k", SIZES)
def test_products(gpu, n, k):
    w = w4.quantize(torch.randn(n, k, device=gpu) * 0.02, 64)
    for rows, dtype in ((1, torch.bfloat16), (4, torch.float16), (5, torch.bfloat16), (16, torch.float16)):
        x, bias = torch.randn(rows, k, device=gpu).to(dtype), torch.randn(n, device=gpu)
        res = torch.randn(rows, n, device=gpu)
        out = w4.linear(x, w, bias=bias, residual=res)
        _check(out, *_reference(x, w, bias=bias, residual=res))
        assert torch.equal(out, w4.linear(x, w, bias=bias, residual=res, out=res.clone()))
