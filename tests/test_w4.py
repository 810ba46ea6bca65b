"""4-bit weights (flashact_amd/w4.py) on the CPU: packing, and the requests that ``linear`` and the C entry refuse."""
import ctypes

import pytest
import torch

from flashact_amd import _lib, w4


@pytest.mark.parametrize("n,k,group", [(1, 8, 32), (16, 128, 128), (33, 136, 64), (5, 1000, 32)])
def test_quantize_takes_the_nearest_value_of_each_group(n, k, group):
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(n + k))
    w[0, :min(k, group)] = 0  # a group of zeros
    p = w4.quantize(w, group)
    assert p["codes"].shape == ((n + 15) // 16, (k + 127) // 128, 4, 16, 16) and p["codes"].dtype == torch.uint8
    assert p["scales"].shape == (p["codes"].shape[0], p["codes"].shape[1] * 128 // group, 16)
    d = w4.dequantize(p)
    assert d.shape == (n, k) and not d[0, :min(k, group)].any()
    grid = torch.tensor(w4.E2M1)
    grid = torch.cat([grid, -grid])
    for i in range(n):
        for g in range(0, k, group):
            x = w[i, g:g + group]
            s = (x.abs().max() / 6).to(torch.bfloat16).float()
            best = ((x[:, None] - grid * s).abs()).amin(1)
            # the chosen value is as near as any, up to the rounding of x / s
            assert ((d[i, g:g + group] - x).abs() <= best + 2 ** -22 * x.abs()).all()


def test_layout_of_codes_and_scales():
    """Byte j of [tile][chunk][q][r] holds columns 128 chunk + 32 (j / 4) + 8 q + 2 (j % 4) and the next."""
    n, k, group = 20, 264, 32
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(1))
    p, d = w4.quantize(w, group), w4.dequantize(w4.quantize(w, group))
    table = torch.tensor(w4.E2M1 + tuple(-v for v in w4.E2M1))
    for i, c in ((0, 0), (3, 37), (16, 255), (19, 263), (7, 130)):
        byte = int(p["codes"][i // 16, c // 128, c % 32 // 8, i % 16, c % 128 // 32 * 4 + c % 8 // 2])
        code = byte >> 4 if c % 2 else byte & 15
        assert float(table[code]) * float(p["scales"][i // 16, c // group, i % 16]) == float(d[i, c])
    assert not p["codes"][1, :, :, 4:].any() and not p["scales"][1, :, 4:].any()  # rows behind the last


def test_quantize_refuses():
    for bad, text in ((torch.randn(4, 12), "multiple of 8"), (torch.randn(4), "multiple of 8"),
                      (torch.full((2, 8), float("nan")), "finite"), (torch.full((2, 8), float("inf")), "finite")):
        with pytest.raises(ValueError, match=text):
            w4.quantize(bad)
    with pytest.raises(ValueError, match="group"):
        w4.quantize(torch.randn(4, 128), 16)


def test_linear_refuses():
    w = w4.quantize(torch.randn(32, 64))
    x = torch.randn(2, 64).bfloat16()
    for kw, err, text in (
            (dict(x=x.float()), TypeError, "bfloat16 or float16"),
            (dict(x=x[:, :32]), ValueError, "K=64"),
            (dict(x=x[None]), ValueError, "K=64"),
            (dict(x=torch.randn(65, 64).bfloat16()), ValueError, "at most 64"),
            (dict(w=dict(w, group=48)), ValueError, "group=48"),
            (dict(w=dict(w, n=33)), ValueError, "codes must be"),
            (dict(w=dict(w, codes=w["codes"].int())), ValueError, "codes must be"),
            (dict(w=dict(w, scales=w["scales"].float())), ValueError, "scales must be"),
            (dict(gate="silu"), ValueError, "gate"),
            (dict(w=w4.quantize(torch.randn(31, 64)), gate="gelu"), ValueError, "even number"),
            (dict(), ValueError, "same GPU"),  # everything right but the device
    ):
        with pytest.raises(err, match=text):
            w4.linear(**{"x": x, "w": w, **kw})


def _args(**kw):
    a = _lib.W4Args()
    fake = 1 << 20  # aligned dummy addresses: validation must fail before anything is dereferenced
    a.x = a.codes = a.scales = a.out = a.workspace = fake
    a.x_stride, a.rows, a.n, a.k, a.group, a.workspace_bytes = 2048, 2, 2560, 2048, 32, 1 << 30
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=1), 1, "dtype"),
    (dict(out_dtype=1), 1, "out_dtype"),
    (dict(rows=65), 1, "rows=65"),
    (dict(rows=-1), 1, "rows=-1"),
    (dict(k=12), 1, "multiple of 8"),
    (dict(n=0), 1, "n=0"),
    (dict(group=16), 1, "group=16"),
    (dict(gate=1, n=33), 1, "even n"),
    (dict(x=None), 1, "x is NULL"),
    (dict(codes=(1 << 20) + 8), 1, "codes is not 16-byte aligned"),
    (dict(residual=(1 << 20) + 2), 1, "residual is not 4-byte aligned"),
    (dict(x_stride=2047), 1, "x_stride"),
    (dict(rows=16, n=2048, k=16384, x_stride=16384, workspace=None, workspace_bytes=0), 1, "workspace"),
])
def test_c_entry_refuses(kw, code, text):
    lib = _lib.lib()
    assert lib.fa_w4_linear(ctypes.byref(_args(**kw)), None) == code
    assert text in lib.fa_last_error().decode()


def test_c_entry_edges():
    lib = _lib.lib()
    assert lib.fa_w4_linear(None, None) == 1
    assert lib.fa_w4_linear(ctypes.byref(_args(rows=0)), None) == 0  # nothing to do, no device needed
    assert lib.fa_w4_workspace_bytes(1, 2560, 2048) == 0 and lib.fa_w4_workspace_bytes(16, 2048, 16384) > 0
    assert lib.fa_w4_workspace_bytes(0, 16, 16) == 0 and lib.fa_w4_workspace_bytes(65, 16, 16) == 0
    if not torch.cuda.is_available():
        assert lib.fa_w4_linear(ctypes.byref(_args()), None) == 3
