"""``w4.linear`` on the MI355X against the product of the dequantised weights in 64 bits.

Tolerance, element by element. The products x * code are exact in fp32; summing K of them with the groups' scales
rounds each step by at most 2^-24 of the running magnitude, so |error| <= (K + K / 32 + 20) 2^-24 sum_k |x W| =: d,
bias and residual among the 20. The result's own rounding adds eps / 2 |y| of its type. Gated: with g and u off by
dg, du and |gelu'| <= 1.13, the error is at most 1.13 dg |u| + |gelu(g)| du + 2^-17 |gelu(g) u|: the device's gelu takes
2^t with t = g (c1 + c3 g^2), three roundings of t (3 2^-24 |t|) and two approximate instructions; where the result
is not lost (|t| < 60) that is below 2^-17 relative.
"""
import math

import pytest
import torch

from flashact_amd import _lib, w4

pytestmark = pytest.mark.gpu

GELU_C = math.sqrt(2 / math.pi)


def _gelu(g):
    return 0.5 * g * (1 + torch.tanh(GELU_C * (g + 0.044715 * g ** 3)))


def _reference(x, w, bias=None, residual=None, gate=None):
    """(result, bound of the fp32 error) in fp64."""
    wd, xd = w4.dequantize(w).double().t().contiguous(), x.double()
    y, k = xd @ wd, w["k"]
    d = (k + k / 32 + 20) * 2.0 ** -24 * (xd.abs() @ wd.abs())
    if bias is not None:
        y, d = y + bias.double(), d + 2.0 ** -24 * bias.double().abs()
    if gate:
        g, u, dg, du = y[..., 0::2], y[..., 1::2], d[..., 0::2], d[..., 1::2]
        y = _gelu(g) * u
        d = 1.13 * dg * u.abs() + _gelu(g).abs() * du + 1.13 * dg * du + 2.0 ** -17 * y.abs()
    if residual is not None:
        y = y + residual.double()
        d = d + 2.0 ** -23 * (y.abs() + residual.double().abs())
    return y, d


def _check(out, ref, bound):
    half = torch.finfo(out.dtype).eps / 2 * (ref.abs() + bound) + torch.finfo(out.dtype).tiny
    err = (out.double() - ref).abs()
    assert bool((err <= bound + half).all()), float((err - bound - half).max())


SHAPES = [(16, 128), (2, 8), (34, 136), (1022, 1000), (2560, 2048), (64, 4104), (4096, 264), (17000, 64)]


@pytest.mark.parametrize("rows", [1, 2, 4, 5, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_products(gpu, rows, dtype):
    gen = torch.Generator(device=gpu).manual_seed(rows)
    for i, (n, k) in enumerate(SHAPES):
        w = w4.quantize(torch.randn(n, k, generator=gen, device=gpu) * 0.02, w4.GROUPS[(i + rows) % 3])
        x = torch.randn(rows, k, generator=gen, device=gpu).to(dtype)
        bias = torch.randn(n, generator=gen, device=gpu)
        res, half = torch.randn(rows, n, generator=gen, device=gpu), torch.randn(rows, n // 2, generator=gen, device=gpu)
        for kw in (dict(), dict(bias=bias), dict(residual=res), dict(gate="gelu"), dict(bias=bias, gate="gelu", residual=half)):
            ref, bound = _reference(x, w, **kw)
            for t in (None, torch.float32):
                out = w4.linear(x, w, out_dtype=t, **kw)
                assert out.dtype == (t or (torch.float32 if "residual" in kw else dtype)) and out.shape == ref.shape
                _check(out, ref, bound)


@pytest.mark.parametrize("group", w4.GROUPS)
def test_odd_rows_of_weights(gpu, group):
    """An odd number of weight rows, and one."""
    for n, k, rows in ((1, 128, 3), (33, 136, 1), (1023, 520, 7), (15, 2048, 20)):
        w = w4.quantize(torch.randn(n, k, device=gpu), group)
        x = torch.randn(rows, k, device=gpu).bfloat16()
        _check(w4.linear(x, w), *_reference(x, w))


def test_long_sums_split_across_workgroups(gpu):
    """K long enough to be split, with and without an epilogue; twice the same bits."""
    for rows, n, k in ((16, 2048, 16384), (1, 48, 16384), (64, 40, 8200), (3, 100, 30000)):
        w = w4.quantize(torch.randn(n, k, device=gpu) * 0.02, 32)
        x, res = torch.randn(rows, k, device=gpu).bfloat16(), torch.randn(rows, n, device=gpu)
        out = w4.linear(x, w, residual=res)
        _check(out, *_reference(x, w, residual=res))
        assert torch.equal(out, w4.linear(x, w, residual=res))


def test_views_in_place_and_single_rows(gpu):
    w = w4.quantize(torch.randn(96, 256, device=gpu), 64)
    wide = torch.randn(5, 1024, device=gpu).bfloat16()
    x = wide[:, 512:768]  # rows with a stride
    assert torch.equal(w4.linear(x, w), w4.linear(x.contiguous(), w))
    assert torch.equal(w4.linear(x[2], w), w4.linear(x, w)[2])  # two chunks: one order of sums
    res = torch.randn(5, 96, device=gpu)
    ref = w4.linear(x, w, residual=res)
    assert w4.linear(x, w, residual=res, out=res) is res and torch.equal(res, ref)
    assert w4.linear(x[:0], w).shape == (0, 96)
    out = torch.full((6, 96), 7.0, device=gpu)
    w4.linear(x, w, out=out[:5])
    assert torch.equal(out[:5], w4.linear(x, w, out_dtype=torch.float32)) and (out[5] == 7).all()


def test_values_that_are_not_numbers_stay_in_their_row(gpu):
    w = w4.quantize(torch.randn(48, 256, device=gpu), 32)
    x = torch.randn(4, 256, device=gpu).bfloat16()
    ref = w4.linear(x, w)
    x[1, 5], x[2, 7] = float("nan"), float("inf")
    out = w4.linear(x, w)
    assert out[1].isnan().all() and not out[2].isfinite().any()
    assert torch.equal(out[0], ref[0]) and torch.equal(out[3], ref[3])



def test_refuses_on_the_gpu(gpu):
    w = w4.quantize(torch.randn(32, 64, device=gpu))
    x = torch.randn(2, 72, device=gpu).bfloat16()
    y, f32 = x[:, :64].contiguous(), torch.zeros(3, 32, device=gpu)
    for kw, err, text in (
            (dict(x=torch.randn(130, device=gpu).bfloat16()[1:65]), ValueError, "aligned"),
            (dict(x=torch.randn(64, 2, device=gpu).bfloat16().t()), ValueError, "contiguous"),
            (dict(x=y[:1].expand(2, 64)), ValueError, "overlap"),
            (dict(bias=torch.randn(32, device=gpu).half()), TypeError, "float32"),
            (dict(bias=torch.randn(31, device=gpu)), ValueError, "bias"),
            (dict(bias=torch.randn(32)), ValueError, "bias"),
            (dict(residual=torch.randn(2, 16, device=gpu)), ValueError, "residual"),
            (dict(out=torch.empty(2, 31, device=gpu)), ValueError, "out must be"),
            (dict(out=torch.empty(2, 32, device=gpu, dtype=torch.int32)), TypeError, "out must be"),
            (dict(out=torch.empty(2, 32, device=gpu), out_dtype=torch.float16), TypeError, "agree"),
            (dict(out=y.view(-1)[:64].view(2, 32)), ValueError, "share memory"),
            (dict(residual=f32[:2], out=f32[1:]), ValueError, "share memory"),
            (dict(out_dtype=torch.float64), TypeError, "out_dtype"),
            (dict(w={k: v.cpu() if torch.is_tensor(v) else v for k, v in w.items()}), ValueError, "same GPU"),
    ):
        with pytest.raises(err, match=text):
            w4.linear(**{"x": y, "w": w, **kw})


def test_split_sums_in_any_workspace(gpu, monkeypatch):
    """The splits' sums meet in memory of any contents: zeros, ones, random words, an earlier call's."""
    x, w = torch.randn(7, 16384, device=gpu).bfloat16(), w4.quantize(torch.randn(2048, 16384, device=gpu) * 0.02, 64)
    ref = w4.linear(x, w)
    need = w4._workspace_bytes(7, 2048, 16384)
    ws = torch.zeros(need, dtype=torch.uint8, device=gpu)
    real = _lib.run_on

    def run_on(index, fn, a, what):
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
        real(index, fn, a, what)

    monkeypatch.setattr(_lib, "run_on", run_on)
    for fill in (None, 0, 255, "random", None, None):
        if fill == "random":
            ws.copy_(torch.randint(0, 256, ws.shape, dtype=torch.uint8, device=gpu))
        elif fill is not None:
            ws.fill_(fill)
        for _ in range(3):
            assert torch.equal(w4.linear(x, w), ref)


@pytest.mark.parametrize("rows,n,k", [(7, 2048, 16384), (1, 64, 16384), (40, 1024, 8192), (20, 512, 4096)])
def test_split_sums_over_the_residual(gpu, rows, n, k):
    """The result takes the residual's place: it is added once, whichever workgroup joins the splits."""
    assert w4._workspace_bytes(rows, n, k) > 0
    x, w = torch.randn(rows, k, device=gpu).bfloat16(), w4.quantize(torch.randn(n, k, device=gpu) * 0.02, 32)
    r = torch.randn(rows, n, device=gpu)
    ref = w4.linear(x, w, residual=r)
    for _ in range(20):
        out = r.clone()
        assert w4.linear(x, w, residual=out, out=out) is out and torch.equal(out, ref)


def test_split_sums_of_inputs_in_turn(gpu):
    """Calls that reuse one another's workspace take no sum of an earlier one."""
    w = w4.quantize(torch.randn(2048, 16384, device=gpu) * 0.02, 32)
    xs = [torch.randn(9, 16384, device=gpu).bfloat16() for _ in range(3)]
    refs = [w4.linear(x, w) for x in xs]
    bad = torch.zeros((), dtype=torch.int64, device=gpu)
    for i in range(600):
        j = (i * 7 + i // 5) % 3
        bad += (w4.linear(xs[j], w) != refs[j]).any()
    assert not torch.equal(refs[0], refs[1]) and bad.item() == 0
