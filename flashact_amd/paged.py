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


# What of a call's checks depends on types, shapes and strides (``_lib.layout``) is done once for each of them, with what follows from
# it for the C call; devices and addresses are looked at in every call. (append with queries: 9.6 us a call so, 12.8 with all of it in each.)
@functools.lru_cache(maxsize=1024)
def _pool_of(k, v, table):
    """(pages, kv_heads, head_dim, samples, pages of a sample, the table's row stride) of layouts, checked."""
    shape = v[1]
    if len(shape) != 5 or shape[2] != PAGE // 8 or shape[4] != 8 or shape[3] not in HEAD_DIMS:
        raise ValueError(f"pool v must be [pages][Hkv][{PAGE // 8}][hd in {HEAD_DIMS}][8], got {tuple(shape)}")
    pages, h, _, hd, _ = shape
    if k[1] != (pages, h, hd // 8, PAGE, 8):
        raise ValueError(f"pool k {tuple(k[1])} does not belong to v {tuple(shape)}")
    t = k[0]
    if (t is not torch.bfloat16 and t is not torch.float16) or v[0] is not t:
        raise TypeError(f"pool k and v must both be bfloat16 or float16, got {t} and {v[0]}")
    if not (_lib.contiguous(k) and _lib.contiguous(v)):
        raise ValueError("pool tensors must be contiguous")
    if not pages * h:
        raise ValueError(f"the pool is empty: {tuple(shape)}")
    tt, ts, tst = table
    if tt is not _I32 or len(ts) != 2 or not ts[0] * ts[1] or (ts[1] > 1 and tst[1] != 1):
        raise ValueError(f"table must be int32 [B][pages of a sample], not empty, rows contiguous, got {tt} {tuple(ts)} with strides {tst}")
    b, width = ts
    stride = tst[0] if b > 1 else width
    if stride < width:
        raise ValueError(f"the table's rows overlap: {tuple(ts)} with strides {tst}")
    return *_lib.ints(pages, h, hd, b, width), stride


def _rows_of(t, k, v, b, h, hd) -> int:
    """The tokens of rows' layouts, checked."""
    if k[0] is not t or v[0] is not t:
        raise TypeError(f"k and v must be {t} like the pool, got {k[0]} and {v[0]}")
    shape = k[1]
    if len(shape) != 4 or shape[0] != b or shape[2] != h or shape[3] != hd or v[1] != shape:
        raise ValueError(f"k and v must be [{b}][tokens][{h}][{hd}], got {tuple(shape)} and {tuple(v[1])}")
    return _lib.ints(shape[1])[0]


def _steps(name, lay) -> tuple:
    """Strides of rows' first three dimensions, for reads of eight dims at once."""
    s = _lib.steps3(lay)
    if lay[2][3] != 1 or s[0] % 8 or s[1] % 8 or s[2] % 8:
        raise ValueError(f"{name} must have contiguous dims and strides that are multiples of 8, got {lay[2]}")
    return s


def _per_sample(name, lay, b):
    if lay is not None and (lay[0] is not _I32 or lay[1] != (b,) or not _lib.contiguous(lay)):
        raise ValueError(f"{name} must be contiguous int32 [{b}], got {lay[0]} {tuple(lay[1])}")


def _on_one(*tensors) -> int:
    """The GPU that all of them (None: none) are on."""
    index = tensors[0].get_device()
    for x in tensors:
        if x is not None and x.get_device() != index:
            index = -1
    if index < 0:
        raise ValueError(f"all tensors must be on one GPU, got {[str(x.device) for x in tensors if x is not None]}")
    return index


@functools.lru_cache(maxsize=1024)
def _append_of(pk, pv, table, k, v, q, start, count, freqs):
    """(strides of q, k and v, the table's row stride, the struct's type and last sizes, the bytes from the first to behind the last
    element of one of the pool's tensors, of k, v and q) of layouts, checked."""
    pages, h, hd, b, width, stride = _pool_of(pk, pv, table)
    tokens = _rows_of(pk[0], k, v, b, h, hd)
    sk, sv, sq, heads = _steps("k", k), _steps("v", v), (0, 0, 0), 0
    if q is not None:
        if q[0] is not pk[0]:
            raise TypeError(f"q must be {pk[0]} like the pool, got {q[0]}")
        if len(q[1]) != 4 or q[1][0] != b or q[1][1] != tokens or q[1][2] < 1 or q[1][3] != hd:
            raise ValueError(f"q must be [{b}][{tokens}][heads][{hd}], got {tuple(q[1])}")
        sq, heads = _steps("q", q), _lib.ints(q[1][2])[0]
    _per_sample("start", start, b)
    _per_sample("count", count, b)
    rotary = 0
    if freqs is not None:
        rotary = 2 * freqs[1][0] if len(freqs[1]) == 1 else -1
        if freqs[0] is not torch.float64 or not 0 < rotary <= hd or rotary % 16 or not _lib.contiguous(freqs):
            raise ValueError(f"freqs must be contiguous float64 [a multiple of 8 up to {hd // 2}], got {freqs[0]} {tuple(freqs[1])}")
    reach = tuple(0 if x is None else 2 * _lib.extent(x) for x in (pk, k, v, q))
    return _S3(*sq), _S4(*sk, 1), _S4(*sv, 1), stride, _lib.DTYPES[pk[0]], (b, tokens, heads, h, hd, pages, width, rotary), reach


def append(pool: dict, table, k, v, start, count=None, *, q=None, freqs=None, adjacent: bool = False):
    """Puts row i < count[b] of k and v (all rows where `count` is None) at token start[b] + i of sample b, in place; returns the
    queries turned alike, where q is given.

    k, v [B][T][Hkv][hd] and q [B][T][H][hd] of the pool's type, strides multiples of 8, dims contiguous; start, count int32 [B].
    freqs (float64, on the GPU, ``frequencies``): keys' and queries' first 2 len(freqs) dims (a multiple of 16) are turned by the
    angles (start[b] + i) freqs[j] on the way, taken in 64 bits; None: nothing is turned. The pairs are dims (j, j + len(freqs)), or
    (2 j, 2 j + 1) with `adjacent` (the packing of ``prefill.pack_backbone``), and become dims (j, j + len(freqs)) in either
    case. Rows behind the table's end or of no page are dropped, as is a sample with a negative start. The result [B][T][H][hd]
    has zeros where a row is not real. Two rows at one token of one page must be ordered by the caller. k, v and q share no memory with the
    pool.
    """
    pk, pv = pool["k"], pool["v"]
    lay = _lib.layout
    sq, sk, sv, stride, dtype, sizes, reach = _append_of(lay(pk), lay(pv), lay(table), lay(k), lay(v), None if q is None else lay(q),
                                                         lay(start), None if count is None else lay(count), None if freqs is None else lay(freqs))
    at_k, at_v, at_q, out, at_out = k.data_ptr(), v.data_ptr(), None if q is None else q.data_ptr(), None, None
    to_k, to_v = pk.data_ptr(), pv.data_ptr()
    whole, *rows = reach
    for at, n in zip((at_k, at_v, at_q or 0), rows):
        if n and (at - whole < to_k < at + n or at - whole < to_v < at + n):
            raise ValueError("k, v and q must not share memory with the pool")
    if (at_k | at_v | (at_q or 0)) % 16:
        raise ValueError("k, v and q must be 16-byte aligned")
    index = _on_one(pk, pv, table, k, v, start, count, q, freqs)
    if q is not None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        at_out = out.data_ptr()
    a = _lib.PagedRowsArgs(dtype, at_q, sq, at_out, at_k, sk, at_v, sv, to_k, to_v, table.data_ptr(), stride,
                           start.data_ptr(), None if count is None else count.data_ptr(), None if freqs is None else freqs.data_ptr(),
                           *sizes, int(adjacent), 0)
    _lib.run_on(index, _lib.lib().fa_paged_append, a, "fa_paged_append")
    return out


def load(pool: dict, table, lens, *, k=None, v=None):
    """Tokens [0, lens[b]) of each sample, as (k, v) rows [B][T][Hkv][hd] of the pool's type.

    Without k and v they are new, of the table's length, with zeros behind lens[b]. Given (any strides, T rows), they are
    written in place up to min(lens[b], T) and left as they are behind it: a view of ``pi05.make_caches`` caches takes a prefix
    to the denoise loop. Tokens of no page are zeros.
    """
    pk, pv = pool["k"], pool["v"]
    pages, h, hd, b, width, stride = _pool_of(_lib.layout(pk), _lib.layout(pv), _lib.layout(table))
    if (k is None) != (v is None):
        raise ValueError("pass both of k and v or neither")
    fresh = k is None
    if fresh:
        shape = (b, width * PAGE, h, hd)
        k, v = pk.new_empty(shape), pk.new_empty(shape)
    tokens = _rows_of(pk.dtype, _lib.layout(k), _lib.layout(v), b, h, hd)
    _per_sample("lens", _lib.layout(lens), b)
    index = _on_one(pk, pv, table, k, v, lens)
    if not fresh:
        if _lib.doubled(k) or _lib.doubled(v) or _lib.meet(k, v):
            raise ValueError("k and v are written: no two of their elements may be one")
        if any(_lib.overlaps(x, (pk, pv, table, lens)) for x in (k, v)):
            raise ValueError("k and v must not share memory with the pool, the table or lens")
    a = _lib.PagedRowsArgs(_lib.DTYPES[pk.dtype], None, _S3(0, 0, 0), None, k.data_ptr(), _S4(*k.stride()), v.data_ptr(),
                           _S4(*v.stride()), pk.data_ptr(), pv.data_ptr(), table.data_ptr(), stride, None,
                           lens.data_ptr(), None, b, tokens, 0, h, hd, pages, width, 0, 0, int(fresh))
    _lib.run_on(index, _lib.lib().fa_paged_load, a, "fa_paged_load")
    return k, v


@functools.lru_cache(maxsize=1024)
def _attend_of(pk, pv, table, q, lens, count, slopes):
    """(the result's shape, strides of q, the table's row stride, the struct's type, its sizes, the workspace's bytes) of layouts, checked."""
    pages, h, hd, b, width, stride = _pool_of(pk, pv, table)
    t, shape = q[0], q[1]
    if t is not pk[0]:
        raise TypeError(f"q must be {pk[0]} like the pool, got {t}")
    if len(shape) != 4 or shape[0] != b or shape[3] != hd or shape[2] < 1 or shape[2] % h:
        raise ValueError(f"q must be [{b}][tokens][a multiple of {h}][{hd}], got {tuple(shape)}")
    steps = _steps("q", q)
    _per_sample("lens", lens, b)
    _per_sample("count", count, b)
    if slopes is not None and (slopes[0] is not _F32 or slopes[1] != (shape[2],) or not _lib.contiguous(slopes)):
        raise ValueError(f"slopes must be contiguous float32 [{shape[2]}], got {slopes[0]} {tuple(slopes[1])}")
    sizes = _lib.ints(b, shape[1], shape[2], h, hd, pages, width)
    need = _workspace_bytes(b, shape[1], shape[2], h, hd, width)
    return tuple(shape), _S3(*steps), stride, _lib.DTYPES[t], sizes, need


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
    pk, pv = pool["k"], pool["v"]
    lay = _lib.layout
    shape, sq, stride, dtype, sizes, need = _attend_of(lay(pk), lay(pv), lay(table), lay(q), lay(lens), None if count is None else lay(count),
                                                       None if slopes is None else lay(slopes))
    if not 0.0 <= softcap < float("inf"):
        raise ValueError(f"softcap must be finite and >= 0, got {softcap}")
    index = _on_one(pk, pv, table, q, lens, count, slopes)
    at = q.data_ptr()
    if at % 16:
        raise ValueError("q must be 16-byte aligned")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.dtype is not q.dtype or out.shape != shape or not out.is_contiguous() or out.get_device() != index or out.data_ptr() % 16:
        raise ValueError(f"out must be contiguous, 16-byte aligned {q.dtype} {shape}, got {out.dtype} {tuple(out.shape)}")
    elif _lib.overlap(out, q) and (out.data_ptr() != at or not q.is_contiguous()):
        raise ValueError("out must not share memory with q but for being it")
    elif _lib.overlaps(out, (pk, pv, table, lens, count, slopes)):
        raise ValueError("out must not share memory with the pool, the table, lens, count or slopes")
    ws = q.new_empty(need // 2) if need else None
    a = _lib.PagedAttnArgs(dtype, at, sq, pk.data_ptr(), pv.data_ptr(), table.data_ptr(), stride, lens.data_ptr(),
                           None if count is None else count.data_ptr(), None if slopes is None else slopes.data_ptr(), *sizes, int(causal),
                           shape[3] ** -0.5 if scale is None else scale, softcap, out.data_ptr(), None if ws is None else ws.data_ptr(), need)
    _lib.run_on(index, _lib.lib().fa_paged_attention, a, "fa_paged_attention")
    return out
