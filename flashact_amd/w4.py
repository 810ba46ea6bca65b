"""Weights in 4 bits on MI355X: packing, and products of a few rows of activations with them (``linear``).

The backbone's decoding form: where a prompt runs through the weights as one large product (``prefill``), tokens
answered one by one read every weight for a handful of rows, and the time is the weights' bytes. Codes are OCP e2m1
with one bf16 scale for each group of 32, 64 or 128 columns, 4.5 bits a weight at a group of 32, next to the 16 of
``pi05.pack_weights`` and the 8 of ``pi05.pack_weights_fp8``. The layout is the kernel's (C ABI ``fa_w4_linear``).
"""
from __future__ import annotations

import functools

import torch

from . import _lib

MAX_ROWS = 64
GROUPS = (32, 64, 128)
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_DT = _lib.DTYPES


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(rows, n, k) -> int:
    """A function of the sizes alone."""
    return _lib.lib().fa_w4_workspace_bytes(rows, n, k)


def quantize(w: torch.Tensor, group: int = 32) -> dict:
    """[N][K] weights -> {"codes", "scales", "n", "k", "group"} as ``linear`` takes them.

    scale = bf16(max|w| / 6) over each group of `group` columns, code = the e2m1 value nearest to w / scale (ties to
    the smaller magnitude); a group of zeros has scale 0. K must be a multiple of 8; rows and columns are padded
    with zeros to the tiles of 16 x 128.
    """
    if w.dim() != 2 or w.shape[0] < 1 or w.shape[1] < 8 or w.shape[1] % 8:
        raise ValueError(f"weights must be [N][K] with K a multiple of 8, got {tuple(w.shape)}")
    if group not in GROUPS:
        raise ValueError(f"group must be one of {GROUPS}, got {group}")
    n, k = w.shape
    nt, kc = (n + 15) // 16, (k + 127) // 128
    w = torch.nn.functional.pad(w.float(), (0, kc * 128 - k, 0, nt * 16 - n))
    if not bool(torch.isfinite(w).all()):
        raise ValueError("weights must be finite")
    g = w.view(nt * 16, -1, group)
    s = (g.abs().amax(-1) / 6.0).to(torch.bfloat16)
    y = torch.where(s[..., None] > 0, g / s.float()[..., None], 0.0).view(nt * 16, kc * 128)
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)
    c = torch.bucketize(y.abs(), edges).to(torch.uint8) | ((y < 0).to(torch.uint8) << 3)
    # [tile, r, chunk, i, q, j, nibble] -> [tile, chunk, q, r, (i, j)]
    c = c.view(nt, 16, kc, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 5, 6)
    codes = (c[..., 0] | (c[..., 1] << 4)).reshape(nt, kc, 4, 16, 16).contiguous()
    scales = s.view(nt, 16, -1).transpose(1, 2).contiguous()
    return {"codes": codes, "scales": scales, "n": n, "k": k, "group": group}


def dequantize(w: dict) -> torch.Tensor:
    """The fp32 weights [N][K] that packed codes and scales stand for."""
    nt, kc = w["codes"].shape[:2]
    c = torch.stack([w["codes"] & 15, w["codes"] >> 4], -1).view(nt, kc, 4, 16, 4, 4, 2).permute(0, 3, 1, 4, 2, 5, 6)
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=c.device)
    x = table[c.reshape(nt * 16, kc * 128).long()]
    s = w["scales"].transpose(1, 2).reshape(nt * 16, -1).float().repeat_interleave(w["group"], 1)
    return (x * s)[:w["n"], :w["k"]]


def linear(x: torch.Tensor, w: dict, *, bias=None, residual=None, gate=None, out=None, out_dtype=None) -> torch.Tensor:
    """x W^T for up to 64 rows of activations, on the current stream.

    x [..][K] bf16 or fp16 (1 or 2 dimensions; rows may be strided); w: a ``quantize`` result. bias [N] fp32 is added
    to the product. gate="gelu": the rows 2f and 2f + 1 of W are a gate and its input (the interleaved packing of
    ``prefill.pack_backbone``), and the result is gelu_tanh(y[2f]) y[2f + 1], of width N / 2. residual fp32, shaped
    like the result, is added last. The result has x's type, or fp32 with a residual, or out's / out_dtype; `out` may be
    the residual itself.
    """
    codes, scales, n, k, group = w["codes"], w["scales"], w["n"], w["k"], w["group"]
    xt = x.dtype
    if xt is not torch.bfloat16 and xt is not torch.float16:
        raise TypeError(f"x must be bfloat16 or float16, got {xt}")
    dim = x.dim()
    if dim not in (1, 2) or x.shape[-1] != k:
        raise ValueError(f"x must be [K={k}] or [rows][K={k}], got {tuple(x.shape)}")
    rows = x.shape[0] if dim == 2 else 1
    if rows > MAX_ROWS:
        raise ValueError(f"{rows} rows: at most {MAX_ROWS} (more rows want a matrix product on unpacked weights)")
    if group not in GROUPS or n < 1 or k < 8 or k % 8:
        raise ValueError(f"weights with n={n}, k={k}, group={group}")
    nt, kc = (n + 15) // 16, (k + 127) // 128
    if codes.dtype is not torch.uint8 or codes.shape != (nt, kc, 4, 16, 16) or not codes.is_contiguous():
        raise ValueError(f"codes must be contiguous uint8 {(nt, kc, 4, 16, 16)}, got {codes.dtype} {tuple(codes.shape)}")
    if scales.dtype is not torch.bfloat16 or scales.shape != (nt, kc * (128 // group), 16) or not scales.is_contiguous():
        raise ValueError(f"scales must be contiguous bfloat16 {(nt, kc * (128 // group), 16)}, got {scales.dtype} "
                         f"{tuple(scales.shape)}")
    if gate is not None and (gate != "gelu" or n % 2):
        raise ValueError(f"gate must be None or 'gelu' (with an even number of weight rows), got {gate!r} and n={n}")
    width = n if gate is None else n // 2
    shape = (rows, width) if dim == 2 else (width,)
    index = x.get_device()
    if index < 0 or codes.get_device() != index or scales.get_device() != index:
        raise ValueError("x, codes and scales must be on the same GPU")
    for name, v, want in (("bias", bias, (n,)), ("residual", residual, shape)):
        if v is not None:
            if v.dtype is not torch.float32:
                raise TypeError(f"{name} must be float32, got {v.dtype}")
            if v.shape != want or not v.is_contiguous() or v.get_device() != index:
                raise ValueError(f"{name} must be contiguous {want} on x's GPU, got {tuple(v.shape)} on {v.device}")
    stride = x.stride(0) if rows > 1 and dim == 2 else k
    if x.stride(-1) != 1 or stride % 8 or stride < k or x.data_ptr() % 16:
        raise ValueError(f"x must have contiguous, 16-byte aligned rows that do not overlap, got strides {x.stride()}")
    if out is None:
        t = out_dtype or (xt if residual is None else torch.float32)
        if t not in _DT:
            raise TypeError(f"out_dtype must be bfloat16, float16 or float32, got {t}")
        out = x.new_empty(shape, dtype=t)
    else:
        t = out.dtype
        if t not in _DT or (out_dtype is not None and out_dtype is not t):
            raise TypeError(f"out must be bfloat16, float16 or float32 and agree with out_dtype, got {t}")
        if out.shape != shape or not out.is_contiguous() or out.get_device() != index:
            raise ValueError(f"out must be contiguous {shape} on x's GPU, got {tuple(out.shape)} on {out.device}")
        being = residual is not None and out.data_ptr() == residual.data_ptr() and t is torch.float32
        if _lib.overlap(out, x) or (residual is not None and not being and _lib.overlap(out, residual)):
            raise ValueError("out must not share memory with x, nor with a residual but for being it")
        if _lib.overlap(out, codes) or _lib.overlap(out, scales) or (bias is not None and _lib.overlap(out, bias)):
            raise ValueError("out must not share memory with the weights or the bias")
    if rows == 0:
        return out
    lib = _lib.lib()
    need = _workspace_bytes(rows, n, k)
    ws = x.new_empty(need, dtype=torch.uint8) if need else None
    a = _lib.W4Args(_DT[xt], _DT[t], x.data_ptr(), stride, codes.data_ptr(), scales.data_ptr(), rows, n, k, group,
                    None if bias is None else bias.data_ptr(), None if residual is None else residual.data_ptr(),
                    0 if gate is None else 1, out.data_ptr(), None if ws is None else ws.data_ptr(), need)
    _lib.run_on(index, lib.fa_w4_linear, a, "fa_w4_linear")
    return out
