"""The paged K/V cache on MI355X: ``append`` rows into it with the position's rotation on the way, ``load`` them back, ``attend``
over it.

Where ``kv8.make_caches`` gives every sample a stretch of its own of one fixed capacity, here all samples draw pages of 32 tokens
from one pool, at the rows' own 16 bits: a request holds as much memory as it has tokens, requests with a common beginning may
share its pages, and a request that ends gives its pages back. A pool is a dict of plain tensors, one layer's: ``k``
[pages][Hkv][hd / 8][32][8] and ``v`` [pages][Hkv][4][hd][8] (token 8 i + j of a page is [i][dim][j]). Which pages are whose is
the caller's: a table, int32 [B][n] on the GPU, names the page of tokens 32 i .. 32 i + 31 of each sample, the same for all
layers; so are the lengths. A captured graph serves every length and every table.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib

PAGE = 32
HEAD_DIMS = (64, 96, 128, 256)
_I32, _F32 = torch.int32, torch.float32
_S3, _S4 = ctypes.c_longlong * 3, ctypes.c_longlong * 4


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(b, tokens, heads, h, hd, width) -> int:
    """A function of the sizes alone."""
    return _lib.lib().fa_paged_attention_workspace_bytes(b, tokens, heads, h, hd, width) if tokens else 0


def make_pools(num_layers: int, pages: int, kv_heads: int = 1, head_dim: int = 256, dtype=torch.bfloat16, device="cuda") -> list:
    """Pools of `num_layers` layers, `pages` pages of 32 tokens each (zeros)."""
    if min(num_layers, pages, kv_heads) < 1 or head_dim not in HEAD_DIMS:
        raise ValueError(f"num_layers={num_layers}, pages={pages}, kv_heads={kv_heads} must be >= 1 and head_dim={head_dim} one of "
                         f"{HEAD_DIMS}")
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError(f"dtype must be bfloat16 or float16, got {dtype}")
    return [{"k": torch.zeros(pages, kv_heads, head_dim // 8, PAGE, 8, dtype=dtype, device=device),
             "v": torch.zeros(pages, kv_heads, PAGE // 8, head_dim, 8, dtype=dtype, device=device)} for _ in range(num_layers)]


def frequencies(dims: int = 256, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """base^(-2 j / dims), j < dims / 2: the angles (radians a position, float64) that ``append`` turns the first `dims` dims by."""
    if dims < 16 or dims % 16 or not 0.0 < base < float("inf"):
        raise ValueError(f"dims={dims} must be a multiple of 16 and base={base} positive")
    return base ** (-torch.arange(0, dims, 2, dtype=torch.float64, device=device) / dims)


def _pool(pool, table):
    """(k, v, pages, kv_heads, head_dim, GPU index, samples, pages of a sample, the table's row stride), checked."""
    k, v = pool["k"], pool["v"]
    shape = v.shape
    if len(shape) != 5 or shape[2] != PAGE // 8 or shape[4] != 8 or shape[3] not in HEAD_DIMS:
        raise ValueError(f"pool v must be [pages][Hkv][{PAGE // 8}][hd in {HEAD_DIMS}][8], got {tuple(shape)}")
    pages, h, _, hd, _ = shape
    if k.shape != (pages, h, hd // 8, PAGE, 8):
        raise ValueError(f"pool k {tuple(k.shape)} does not belong to v {tuple(shape)}")
    t = k.dtype
    if (t is not torch.bfloat16 and t is not torch.float16) or v.dtype is not t:
        raise TypeError(f"pool k and v must both be bfloat16 or float16, got {t} and {v.dtype}")
    if not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("pool tensors must be contiguous")
    if not pages * h:
        raise ValueError(f"the pool is empty: {tuple(shape)}")
    index = v.get_device()
    if (table.dtype is not _I32 or table.dim() != 2 or table.get_device() != index or not table.numel()
            or (table.shape[1] > 1 and table.stride(1) != 1)):
        raise ValueError(f"table must be int32 [B][pages of a sample], not empty, rows contiguous, on the pool's GPU, got {table.dtype} "
                         f"{tuple(table.shape)} on {table.device}")
    if k.get_device() != index:
        raise ValueError("the pool's tensors must be on one GPU")
    b, width = table.shape
    stride = table.stride(0) if b > 1 else width
    if stride < width:
        raise ValueError(f"the table's rows overlap: {tuple(table.shape)} with strides {table.stride()}")
    return k, v, pages, h, hd, index, b, width, stride


def _index(name, t, b, index):
    if t.dtype is not _I32 or t.shape != (b,) or not t.is_contiguous() or t.get_device() != index:
        raise ValueError(f"{name} must be contiguous int32 [{b}] on the pool's GPU, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(pk, k, v, b, h, hd, index):
    """The rows' tokens, checked."""
    if k.dtype is not pk.dtype or v.dtype is not pk.dtype:
        raise TypeError(f"k and v must be {pk.dtype} like the pool, got {k.dtype} and {v.dtype}")
    shape = k.shape
    if len(shape) != 4 or shape[0] != b or shape[2] != h or shape[3] != hd or v.shape != shape:
        raise ValueError(f"k and v must be [{b}][tokens][{h}][{hd}], got {tuple(shape)} and {tuple(v.shape)}")
    if index < 0 or k.get_device() != index or v.get_device() != index:
        raise ValueError(f"pool, k and v must be on the same GPU, got {k.device} and {v.device}")
    return shape[1]


def append(pool: dict, table, k, v, start, count=None, *, q=None, freqs=None, adjacent: bool = False):
    """Puts row i < count[b] of k and v (all rows where `count` is None) at token start[b] + i of sample b, in place; returns the
    queries turned alike, where q is given.

    k, v [B][T][Hkv][hd] and q [B][T][H][hd] of the pool's type, strides multiples of 8, dims contiguous; start, count int32 [B].
    freqs (float64, on the GPU, ``frequencies``): keys' and queries' first 2 len(freqs) dims (a multiple of 16) are turned by the
    angles (start[b] + i) freqs[j] on the way, taken in 64 bits; None: nothing is turned. The pairs are dims (j, j + len(freqs)), or
    (2 j, 2 j + 1) with `adjacent` (the packing of ``prefill.pack_backbone``), and become dims (j, j + len(freqs)) in either
    case. Rows behind the table's end or of no page are dropped, as is a sample with a negative start. The result [B][T][H][hd]
    has zeros where a row is not real. Two rows at one token of one page must be ordered by the caller; rows and pool share no memory.
    """
    pk, pv, pages, h, hd, index, b, width, stride = _pool(pool, table)
    tokens = _rows(pk, k, v, b, h, hd, index)
    t = pk.dtype
    sk, sv, sq, heads, out = _lib.strides3(k), _lib.strides3(v), (0, 0, 0), 0, None
    for s, x in ((sk, k), (sv, v)):
        if x.stride(3) != 1 or s[0] % 8 or s[1] % 8 or s[2] % 8 or x.data_ptr() % 16:
            raise ValueError("k and v must have contiguous dims and strides that are multiples of 8, 16-byte aligned, got "
                             f"{x.stride()}")
    if q is not None:
        if q.dtype is not t:
            raise TypeError(f"q must be {t} like the pool, got {q.dtype}")
        if q.dim() != 4 or q.shape[0] != b or q.shape[1] != tokens or q.shape[2] < 1 or q.shape[3] != hd:
            raise ValueError(f"q must be [{b}][{tokens}][heads][{hd}], got {tuple(q.shape)}")
        sq, heads = _lib.strides3(q), q.shape[2]
        if q.stride(3) != 1 or sq[0] % 8 or sq[1] % 8 or sq[2] % 8 or q.data_ptr() % 16 or q.get_device() != index:
            raise ValueError("q must have contiguous dims and strides that are multiples of 8, 16-byte aligned, on the pool's GPU, got "
                             f"{q.stride()} on {q.device}")
        out = q.new_empty((b, tokens, heads, hd))
    rotary = 0
    if freqs is not None:
        rotary = 2 * freqs.shape[0] if freqs.dim() == 1 else -1
        if (freqs.dtype is not torch.float64 or not 0 < rotary <= hd or rotary % 16 or not freqs.is_contiguous()
                or freqs.get_device() != index):
            raise ValueError(f"freqs must be contiguous float64 [a multiple of 8 up to {hd // 2}] on the pool's GPU, got {freqs.dtype} "
                             f"{tuple(freqs.shape)} on {freqs.device}")
    a = _lib.PagedRowsArgs(_lib.DTYPES[t], None if q is None else q.data_ptr(), _S3(*sq), None if out is None else out.data_ptr(),
                           k.data_ptr(), _S4(*sk, 1), v.data_ptr(), _S4(*sv, 1), pk.data_ptr(), pv.data_ptr(), table.data_ptr(),
                           stride, _index("start", start, b, index), None if count is None else _index("count", count, b, index),
                           None if freqs is None else freqs.data_ptr(), b, tokens, heads, h, hd, pages, width, rotary,
                           int(adjacent), 0)
    _lib.run_on(index, _lib.lib().fa_paged_append, a, "fa_paged_append")
    return out


def load(pool: dict, table, lens, *, k=None, v=None):
    """Tokens [0, lens[b]) of each sample, as (k, v) rows [B][T][Hkv][hd] of the pool's type.

    Without k and v they are new, of the table's length, with zeros behind lens[b]. Given (any strides, T rows), they are
    written in place up to min(lens[b], T) and left as they are behind it: a view of ``pi05.make_caches`` caches takes a prefix
    to the denoise loop. Tokens of no page are zeros.
    """
    pk, pv, pages, h, hd, index, b, width, stride = _pool(pool, table)
    if (k is None) != (v is None):
        raise ValueError("pass both of k and v or neither")
    fresh = k is None
    if fresh:
        shape = (b, width * PAGE, h, hd)
        k, v = pk.new_empty(shape), pk.new_empty(shape)
    tokens = _rows(pk, k, v, b, h, hd, index)
    if not fresh:
        if _lib.doubled(k) or _lib.doubled(v) or _lib.meet(k, v):
            raise ValueError("k and v are written: no two of their elements may be one")
        if any(_lib.overlap(x, y) for x in (k, v) for y in (pk, pv, table, lens)):
            raise ValueError("k and v must not share memory with the pool, the table or lens")
    a = _lib.PagedRowsArgs(_lib.DTYPES[pk.dtype], None, _S3(0, 0, 0), None, k.data_ptr(), _S4(*k.stride()), v.data_ptr(),
                           _S4(*v.stride()), pk.data_ptr(), pv.data_ptr(), table.data_ptr(), stride, None,
                           _index("lens", lens, b, index), None, b, tokens, 0, h, hd, pages, width, 0, 0, int(fresh))
    _lib.run_on(index, _lib.lib().fa_paged_load, a, "fa_paged_load")
    return k, v


def attend(q, pool: dict, table, lens, *, count=None, scale=None, softcap: float = 0.0, slopes=None, causal: bool = True,
           out=None) -> torch.Tensor:
    """Attention of each sample's newest tokens over its pages (they themselves appended before the call).

    q [B][T][H][hd] of the pool's type (H a multiple of its heads; strides multiples of 8, dims contiguous); lens int32
    [B]: cached tokens (those behind the table's end do not count); count int32 [B]: how many of the T are real (None: all). Query
    t < n is at position i = lens - n + t and sees keys j <= i, or all of the cached ones with causal=False; keys of no page are
    not seen. Scores are q . k * scale (default hd^-1/2), capped to softcap * tanh(s / softcap) where softcap > 0, less
    slopes[h] |i - j| where slopes (fp32 [H]) are given. Rows without keys become zero; what a row does not see never reaches it, and
    an infinite value that it sees leaves that dim infinite or NaN. Returns [B][T][H][hd] of q's type, in
    `out` where it is given (q itself may be).
    """
    pk, pv, pages, h, hd, index, b, width, stride = _pool(pool, table)
    t = pk.dtype
    if q.dtype is not t:
        raise TypeError(f"q must be {t} like the pool, got {q.dtype}")
    if q.dim() != 4 or q.shape[0] != b or q.shape[3] != hd or q.shape[2] < 1 or q.shape[2] % h:
        raise ValueError(f"q must be [{b}][tokens][a multiple of {h}][{hd}], got {tuple(q.shape)}")
    tokens, heads = q.shape[1], q.shape[2]
    sb, st, sh = _lib.strides3(q)
    if q.stride(3) != 1 or sb % 8 or st % 8 or sh % 8 or q.data_ptr() % 16:
        raise ValueError(f"q must have contiguous dims and strides that are multiples of 8, 16-byte aligned, got {q.stride()}")
    softcap = float(softcap)
    if not 0.0 <= softcap < float("inf"):
        raise ValueError(f"softcap must be finite and >= 0, got {softcap}")
    if index < 0 or q.get_device() != index:
        raise ValueError(f"pool and q must be on the same GPU, got {q.device}")
    if slopes is not None and (slopes.dtype is not _F32 or slopes.shape != (heads,) or not slopes.is_contiguous()
                               or slopes.get_device() != index):
        raise ValueError(f"slopes must be contiguous float32 [{heads}] on q's GPU, got {slopes.dtype} {tuple(slopes.shape)}")
    if out is None:
        out = q.new_empty((b, tokens, heads, hd))
    elif out.dtype is not t or out.shape != q.shape or not out.is_contiguous() or out.get_device() != index or out.data_ptr() % 16:
        raise ValueError(f"out must be contiguous, 16-byte aligned {t} {tuple(q.shape)}, got {out.dtype} {tuple(out.shape)}")
    elif _lib.overlap(out, q) and (out.data_ptr() != q.data_ptr() or not q.is_contiguous()):
        raise ValueError("out must not share memory with q but for being it")
    elif any(x is not None and _lib.overlap(out, x) for x in (pk, pv, table, lens, count, slopes)):
        raise ValueError("out must not share memory with the pool, the table, lens, count or slopes")
    need = _workspace_bytes(b, tokens, heads, h, hd, width)
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    a = _lib.PagedAttnArgs(_lib.DTYPES[t], q.data_ptr(), _S3(sb, st, sh), pk.data_ptr(), pv.data_ptr(), table.data_ptr(), stride,
                           _index("lens", lens, b, index), None if count is None else _index("count", count, b, index),
                           None if slopes is None else slopes.data_ptr(), b, tokens, heads, h, hd, pages, width, int(causal),
                           hd ** -0.5 if scale is None else scale, softcap, out.data_ptr(), None if ws is None else ws.data_ptr(),
                           need)
    _lib.run_on(index, _lib.lib().fa_paged_attention, a, "fa_paged_attention")
    return out
