"""Low-rank adapters of many requests at once on MI355X: ``pack`` them into a bank, ``add`` each row's own to a shared projection.

One backbone serves several fine-tuned tasks: the large projections (``w4.linear``, or a matrix product over a prompt) are the
same for all rows of a batch, and each row adds scale B (A x) of the adapter that its request names, or nothing. A bank is a dict
of plain tensors, one projection's: ``a`` [adapters][K / 8][rank][8], ``b`` [adapters][rank / 8][N][8] and ``scale`` [adapters]
fp32, the layout of the kernels (C ABI ``fa_lora_add``).
"""
from __future__ import annotations

import functools

import torch

from . import _lib

MAX_RANK = 128
_DT = _lib.DTYPES


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(rows, k, rank) -> int:
    """A function of the sizes alone."""
    return _lib.lib().fa_lora_workspace_bytes(rows, k, rank)


def pack(adapters: list, dtype=torch.bfloat16) -> dict:
    """A bank of adapters (A [rank][K], B [N][rank], scale), whose ranks may differ: they are padded with zeros to the largest,
    rounded up to a multiple of 8. K must be a multiple of 8."""
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError(f"dtype must be bfloat16 or float16, got {dtype}")
    if not adapters:
        raise ValueError("a bank needs an adapter")
    n, k = adapters[0][1].shape[0], adapters[0][0].shape[-1]
    for a, b, _ in adapters:
        if a.dim() != 2 or b.dim() != 2 or a.shape[1] != k or b.shape[0] != n or a.shape[0] != b.shape[1] or not 0 < a.shape[0] <= MAX_RANK:
            raise ValueError(f"adapters must be A [rank][{k}] and B [{n}][rank] of ranks up to {MAX_RANK}, got {tuple(a.shape)} and "
                             f"{tuple(b.shape)}")
    if k % 8 or not n * k:
        raise ValueError(f"K={k} must be a multiple of 8, and N={n} not 0")
    rank = (max(a.shape[0] for a, _, _ in adapters) + 7) // 8 * 8
    pad = torch.nn.functional.pad
    a = torch.stack([pad(a, (0, 0, 0, rank - a.shape[0])).to(dtype) for a, _, _ in adapters])
    b = torch.stack([pad(b, (0, rank - b.shape[1])).to(dtype) for _, b, _ in adapters])
    if not (bool(torch.isfinite(a).all()) and bool(torch.isfinite(b).all())):
        raise ValueError("adapters must be finite")
    return {"a": a.view(-1, rank, k // 8, 8).transpose(1, 2).contiguous(), "b": b.view(-1, n, rank // 8, 8).transpose(1, 2).contiguous(),
            "scale": torch.tensor([float(s) for _, _, s in adapters], dtype=torch.float32, device=a.device)}


def unpack(bank: dict) -> list:
    """The adapters (A [rank][K], B [N][rank], scale) of a bank, as views and host numbers."""
    return [(a.transpose(0, 1).flatten(1), b.transpose(0, 1).flatten(1), s) for a, b, s in zip(bank["a"], bank["b"], bank["scale"].tolist())]


@functools.lru_cache(maxsize=1024)
def _add_of(y, x, a, b, scale, index, gate):
    """(the struct's types, the result's shape and type, x's row stride, the struct's sizes, the workspace's bytes, 0 without rows) of
    layouts (``_lib.layout``), checked: done once for each of them."""
    t, sx, stx = x
    if t is not torch.bfloat16 and t is not torch.float16:
        raise TypeError(f"x must be bfloat16 or float16, got {t}")
    if a[0] is not t or b[0] is not t or scale[0] is not torch.float32:
        raise TypeError(f"the bank's a and b must be {t} like x and scale float32, got {a[0]}, {b[0]} and {scale[0]}")
    if y[0] is not t and y[0] is not torch.float32:
        raise TypeError(f"y must be float32 or {t} like x, got {y[0]}")
    sa, sb = a[1], b[1]
    if (len(sa) != 4 or len(sb) != 4 or sa[3] != 8 or sb[3] != 8 or sa[0] != sb[0] or sa[2] != 8 * sb[1] or not 0 < sa[2] <= MAX_RANK
            or not sa[0] * sa[1] * sb[2] or scale[1] != sa[:1]):
        raise ValueError(f"the bank must be a [adapters][K / 8][rank][8], b [adapters][rank / 8][N][8] and scale [adapters] with ranks up "
                         f"to {MAX_RANK}, got {tuple(sa)}, {tuple(sb)} and {tuple(scale[1])}")
    if not (_lib.contiguous(a) and _lib.contiguous(b) and _lib.contiguous(scale)):
        raise ValueError("the bank's tensors must be contiguous")
    k, n, rank = 8 * sa[1], sb[2], sa[2]
    rows = sx[0] if len(sx) == 2 else -1
    if rows < 0 or sx[1] != k or y[1] != (rows, n) or index[1] != (rows,):
        raise ValueError(f"x must be [rows][K={k}], y [rows][N={n}] and index [rows], got {tuple(sx)}, {tuple(y[1])} and {tuple(index[1])}")
    if max(n, k) > 1 << 24 or rows > 1 << 20:
        raise ValueError(f"N={n} and K={k} must be at most 2^24 and rows={rows} at most 2^20")
    if index[0] is not torch.int32 or not _lib.contiguous(index) or not _lib.contiguous(y):
        raise ValueError(f"index must be contiguous int32 and y contiguous, got {index[0]} and strides {y[2]}")
    if gate is not None and (gate != "gelu" or n % 2):
        raise ValueError(f"gate must be None or 'gelu' (with an even N), got {gate!r} and N={n}")
    stride = stx[0] if rows > 1 else k
    if stx[1] != 1 or stride % 8 or stride < k:
        raise ValueError(f"x must have contiguous rows that do not overlap, strides multiples of 8, got strides {stx}")
    shape, dt = ((rows, n), y[0]) if gate is None else ((rows, n // 2), t)
    return ((_DT[t], _DT[y[0]]), shape, dt, stride, (rows, n, k, rank, sa[0], 0 if gate is None else 1),
            _workspace_bytes(rows, k, rank) if rows else 0)


def add(y: torch.Tensor, x: torch.Tensor, bank: dict, index: torch.Tensor, *, gate=None, out=None) -> torch.Tensor:
    """y + scale[i] B_i A_i x, row by row with i = index[row]; rows whose index is no adapter's (-1) keep y. On the current stream.

    y [rows][N] contiguous, fp32 or x's type: the shared projection of x [rows][K] bf16 or fp16 (rows may be strided); bank: a
    ``pack`` result of x's type; index int32 [rows] on the GPU. gate="gelu": columns 2f and 2f + 1 of the sum are a gate and its
    input (the interleaved packing of ``prefill.pack_backbone``), and the result is gelu_tanh(sum[2f]) sum[2f + 1], [rows][N / 2] of x's
    type. Else it is like y, in `out` where that is given (y itself may be). An adapter reaches its own rows only.
    """
    a, b, scale = bank["a"], bank["b"], bank["scale"]
    lay = _lib.layout
    dtype, shape, dt, stride, sizes, need = _add_of(lay(y), lay(x), lay(a), lay(b), lay(scale), lay(index), gate)
    at = x.data_ptr()
    if at % 16:
        raise ValueError("x must be 16-byte aligned")
    gpu = x.get_device()
    if not gpu == a.get_device() == b.get_device() == scale.get_device() == y.get_device() == index.get_device() or gpu < 0:
        raise ValueError("x, y, index and the bank must be on the same GPU")
    if out is None:
        out = torch.empty_like(y) if gate is None else x.new_empty(shape)
    elif out.dtype is not dt or out.shape != shape or not out.is_contiguous() or out.get_device() != gpu:
        raise ValueError(f"out must be contiguous {dt} {shape} on x's GPU, got {out.dtype} {tuple(out.shape)} on {out.device}")
    elif (gate is not None or out is not y) and _lib.overlap(out, y) and (gate is not None or out.data_ptr() != y.data_ptr()):
        raise ValueError("out must not share memory with y but for being it, without a gate")
    elif _lib.overlaps(out, (x, a, b, scale, index)):
        raise ValueError("out must not share memory with x, index or the bank")
    if not sizes[0]:
        return out
    ws = x.new_empty(need // 2)
    args = _lib.LoraArgs(*dtype, at, stride, a.data_ptr(), b.data_ptr(), scale.data_ptr(), index.data_ptr(), *sizes, y.data_ptr(),
                         out.data_ptr(), ws.data_ptr(), need)
    _lib.run_on(gpu, _lib.lib().fa_lora_add, args, "fa_lora_add")
    return out
