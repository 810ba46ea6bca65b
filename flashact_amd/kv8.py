"""The 8-bit K/V cache on MI355X: ``store`` rows into it, ``load`` them back, ``attend`` over it.

Where ``pi05.make_caches`` keeps a prefix of one common length in bf16, this cache holds samples of different lengths
at half the bytes and grows token by token: e4m3 codes with one scale for each block of 32 tokens and head, a power
of two, so that a code's rounding (half a step of 2^-3) is the only one. A cache is a dict of plain tensors, one layer's:
``k`` [B][Hkv][blocks][hd / 16][32][16] and ``v`` [B][Hkv][blocks][hd][32] uint8, ``ks`` and ``vs`` [B][Hkv][blocks]
fp32. How many tokens of it count is the caller's, an int32 tensor on the GPU, so a captured graph serves every length.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib

BLOCK = 32
HEAD_DIMS = (64, 96, 128, 256)
_U8, _I32, _F32 = torch.uint8, torch.int32, torch.float32
_S3, _S4 = ctypes.c_longlong * 3, ctypes.c_longlong * 4


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(b, tokens, heads, h, hd, nb) -> int:
    """A function of the sizes alone."""
    return _lib.lib().fa_kv8_attention_workspace_bytes(b, tokens, heads, h, hd, nb) if tokens else 0


def make_caches(num_layers: int, batch: int, max_tokens: int, kv_heads: int = 1, head_dim: int = 256, device="cuda") -> list:
    """Empty caches of `num_layers` layers for up to `max_tokens` tokens (rounded up to blocks of 32) of each sample."""
    if min(num_layers, batch, max_tokens, kv_heads) < 1 or head_dim not in HEAD_DIMS:
        raise ValueError(f"num_layers={num_layers}, batch={batch}, max_tokens={max_tokens}, kv_heads={kv_heads} must be "
                         f">= 1 and head_dim={head_dim} one of {HEAD_DIMS}")
    nb = (max_tokens + BLOCK - 1) // BLOCK
    code = lambda *s: torch.zeros(batch, kv_heads, nb, *s, dtype=torch.uint8, device=device)  # noqa: E731
    unit = lambda: torch.ones(batch, kv_heads, nb, dtype=torch.float32, device=device)  # noqa: E731
    return [{"k": code(head_dim // 16, BLOCK, 16), "v": code(head_dim, BLOCK), "ks": unit(), "vs": unit()}
            for _ in range(num_layers)]


def _cache(cache):
    """(k, v, ks, vs, batch, kv_heads, blocks, head_dim, GPU index) of a cache, checked."""
    k, v, ks, vs = cache["k"], cache["v"], cache["ks"], cache["vs"]
    shape = v.shape
    if len(shape) != 5 or shape[4] != BLOCK or shape[3] not in HEAD_DIMS:
        raise ValueError(f"cache v must be [B][Hkv][blocks][hd in {HEAD_DIMS}][{BLOCK}], got {tuple(shape)}")
    b, h, nb, hd, _ = shape
    units = (b, h, nb)
    if k.shape != (b, h, nb, hd // 16, BLOCK, 16) or ks.shape != units or vs.shape != units:
        raise ValueError(f"cache k {tuple(k.shape)}, ks {tuple(ks.shape)}, vs {tuple(vs.shape)} do not belong to v "
                         f"{tuple(v.shape)}")
    if k.dtype is not _U8 or v.dtype is not _U8 or ks.dtype is not _F32 or vs.dtype is not _F32:
        raise TypeError("cache k and v must be uint8, ks and vs float32")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("cache tensors must be contiguous")
    if not b * h * nb:
        raise ValueError(f"the cache is empty: {tuple(shape)}")
    index = v.get_device()
    if k.get_device() != index or ks.get_device() != index or vs.get_device() != index:
        raise ValueError("the cache's tensors must be on one GPU")
    return k, v, ks, vs, b, h, nb, hd, index


def _index(name, t, b, index):
    if t.dtype is not _I32 or t.shape != (b,) or not t.is_contiguous() or t.get_device() != index:
        raise ValueError(f"{name} must be contiguous int32 [{b}] on the cache's GPU, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(k, v, b, h, hd, index):
    """The rows' tokens and FA_DTYPE, checked."""
    t = _lib.DTYPES.get(k.dtype)
    if t is None or v.dtype is not k.dtype:
        raise TypeError(f"k and v must both be bfloat16, float16 or float32, got {k.dtype} and {v.dtype}")
    shape = k.shape
    if len(shape) != 4 or shape[0] != b or shape[2] != h or shape[3] != hd or v.shape != shape:
        raise ValueError(f"k and v must be [{b}][tokens][{h}][{hd}], got {tuple(shape)} and {tuple(v.shape)}")
    if index < 0 or k.get_device() != index or v.get_device() != index:
        raise ValueError(f"cache, k and v must be on the same GPU, got {k.device} and {v.device}")
    return shape[1], t


def store(cache: dict, k, v, start, count=None) -> None:
    """Puts row i < count[b] of k and v (all rows where `count` is None) at token start[b] + i of sample b, in place.

    k, v [B][T][Hkv][hd] bf16, fp16 or fp32, of any strides; start, count int32 [B]. A block's scale is the smallest
    power of two s with max|x| <= 448 s over its new rows, or that of the block's earlier tokens (before start[b]) if that
    is larger; if it grows they are recoded. Infinities and NaN are stored as NaN and set no scale. Tokens behind the
    new ones keep their codes; rows that do not fit into the cache are dropped, all of a sample whose start is negative.
    """
    ck, cv, ks, vs, b, h, nb, hd, index = _cache(cache)
    tokens, t = _rows(k, v, b, h, hd, index)
    a = _lib.Kv8RowsArgs(t, k.data_ptr(), _S4(*k.stride()), v.data_ptr(), _S4(*v.stride()), ck.data_ptr(),
                         cv.data_ptr(), ks.data_ptr(), vs.data_ptr(), _index("start", start, b, index),
                         None if count is None else _index("count", count, b, index), b, tokens, h, hd, nb, 0)
    _lib.run_on(index, _lib.lib().fa_kv8_store, a, "fa_kv8_store")


def load(cache: dict, lens, *, k=None, v=None, dtype=torch.bfloat16):
    """The values of tokens [0, lens[b]) of each sample, as (k, v) rows [B][T][Hkv][hd].

    Without k and v they are new, of the cache's length and `dtype`, with zeros behind lens[b]. Given (any strides, T
    rows), they are written in place up to min(lens[b], T) and left as they are behind it: a view of
    ``pi05.make_caches`` caches takes a prefix to the denoise loop.
    """
    ck, cv, ks, vs, b, h, nb, hd, index = _cache(cache)
    if (k is None) != (v is None):
        raise ValueError("pass both of k and v or neither")
    fresh = k is None
    if not fresh and (_lib.doubled(k) or _lib.doubled(v) or k.dtype is v.dtype and _lib.meet(k, v)):
        raise ValueError("k and v are written: no two of their elements may be one")
    if fresh:
        if dtype not in _lib.DTYPES:
            raise TypeError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
        shape = (b, nb * BLOCK, h, hd)
        k, v = ck.new_empty(shape, dtype=dtype), ck.new_empty(shape, dtype=dtype)
    tokens, t = _rows(k, v, b, h, hd, index)
    a = _lib.Kv8RowsArgs(t, k.data_ptr(), _S4(*k.stride()), v.data_ptr(), _S4(*v.stride()), ck.data_ptr(),
                         cv.data_ptr(), ks.data_ptr(), vs.data_ptr(), None, _index("lens", lens, b, index), b, tokens, h, hd,
                         nb, int(fresh))
    _lib.run_on(index, _lib.lib().fa_kv8_load, a, "fa_kv8_load")
    return k, v


def attend(q, cache: dict, lens, *, count=None, scale=None, softcap: float = 0.0, slopes=None, causal: bool = True,
           out=None) -> torch.Tensor:
    """Attention of each sample's newest tokens over its cached ones (they themselves stored before the call).

    q [B][T][H][hd] bf16 or fp16 (H a multiple of the cache's heads; strides multiples of 8, dims contiguous); lens int32
    [B]: cached tokens; count int32 [B]: how many of the T are real (None: all). Query t < n is at position
    i = lens - n + t and sees keys j <= i, or all of the cached ones with causal=False. Scores are q . k * scale (default
    hd^-1/2), capped to softcap * tanh(s / softcap) where softcap > 0, less slopes[h] |i - j| where slopes (fp32 [H]) are
    given. Rows without keys become zero. Returns [B][T][H][hd] of q's type, in `out` where it is given (q itself may be).
    """
    ck, cv, ks, vs, b, h, nb, hd, index = _cache(cache)
    if q.dtype is not torch.bfloat16 and q.dtype is not torch.float16:
        raise TypeError(f"q must be bfloat16 or float16, got {q.dtype}")
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
        raise ValueError(f"cache and q must be on the same GPU, got {q.device}")
    if slopes is not None and (slopes.dtype is not torch.float32 or slopes.shape != (heads,) or not slopes.is_contiguous()
                               or slopes.get_device() != index):
        raise ValueError(f"slopes must be contiguous float32 [{heads}] on q's GPU, got {slopes.dtype} {tuple(slopes.shape)}")
    if out is None:
        out = q.new_empty((b, tokens, heads, hd))
    elif out.dtype is not q.dtype or out.shape != q.shape or not out.is_contiguous() or out.get_device() != index:
        raise ValueError(f"out must be contiguous {q.dtype} {tuple(q.shape)}, got {out.dtype} {tuple(out.shape)}")
    elif _lib.overlap(out, q) and (out.data_ptr() != q.data_ptr() or not q.is_contiguous()):
        raise ValueError("out must not share memory with q but for being it")
    elif any(t is not None and _lib.overlap(out, t) for t in (ck, cv, ks, vs, lens, count, slopes)):
        raise ValueError("out must not share memory with the cache, lens, count or slopes")
    lib = _lib.lib()
    need = _workspace_bytes(b, tokens, heads, h, hd, nb)
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    a = _lib.Kv8AttnArgs(_lib.DTYPES[q.dtype], q.data_ptr(), _S3(sb, st, sh), ck.data_ptr(), cv.data_ptr(), ks.data_ptr(),
                         vs.data_ptr(), _index("lens", lens, b, index), None if count is None else _index("count", count, b, index),
                         None if slopes is None else slopes.data_ptr(), b, tokens, heads, h, hd, nb, int(causal),
                         hd ** -0.5 if scale is None else scale, softcap, out.data_ptr(), None if ws is None else ws.data_ptr(),
                         need)
    _lib.run_on(index, lib.fa_kv8_attention, a, "fa_kv8_attention")
    return out
