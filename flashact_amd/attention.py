"""Attention on MI355X in which every query has its own span of keys: ``attend``, and ``prefix_spans`` that makes spans.

The prompt's form of attention for what the prefill's fused kernel does not take: prompts of different lengths packed one
behind the other, a prefix that all of a document sees with causal tokens behind it (the attention pattern of PaliGemma's
prompts, where images and instruction see each other and the answer is causal), capped scores, a distance bias, rows that
are padding. One HIP launch (C ABI ``fa_span_attention``); a second joins the parts where few queries see very many keys.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib

_S3 = ctypes.c_longlong * 3


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(b, tq, tk, heads, hd) -> int:
    """A function of the sizes alone."""
    return _lib.lib().fa_span_attention_workspace_bytes(b, tq, tk, heads, hd)


def prefix_spans(lengths, prefix, total: int) -> torch.Tensor:
    """Spans [total][2] (int32, on the lengths' device) of documents packed one behind the other in `total` rows.

    lengths, prefix: integer [N]: tokens of each document, and how many of its first ones all of it sees (0: causal, the
    document's length: no mask in it). Token i of a document sees its tokens 0 .. max(i, prefix - 1). Rows behind the last
    document see nothing. No host synchronisation; documents that pass `total` are cut off.
    """
    if lengths.dim() != 1 or prefix.shape != lengths.shape or lengths.is_floating_point() or prefix.is_floating_point():
        raise ValueError(f"lengths and prefix must be integer [N], got {tuple(lengths.shape)} and {tuple(prefix.shape)}")
    if total < 0:
        raise ValueError(f"total must be >= 0, got {total}")
    row = torch.arange(total, device=lengths.device)
    if lengths.shape[0] == 0:
        return torch.zeros(total, 2, dtype=torch.int32, device=lengths.device)
    n = lengths.long().clamp(min=0)
    end = n.cumsum(0)
    doc = torch.searchsorted(end, row, right=True)
    there = doc < n.shape[0]
    doc = doc.clamp(max=n.shape[0] - 1)
    first = (end - n)[doc]
    last = torch.maximum(row + 1, first + torch.minimum(prefix.long(), n)[doc])
    spans = torch.stack([first, last.clamp(max=total)], -1)
    return torch.where(there[:, None], spans, 0).to(torch.int32)


def attend(q, k, v, spans=None, *, scale=None, softcap: float = 0.0, slopes=None, out=None) -> torch.Tensor:
    """Attention of every query over its own span of keys, on the current stream; [B][Tq][H][hd] of q's type.

    q [B][Tq][H][hd], k and v [B][Tk][Hkv][hd] bf16 or fp16, H a multiple of Hkv, hd a multiple of 8 up to 256; strides
    multiples of 8, dims contiguous. spans int32 [B][Tq][2] (or [Tq][2] for all samples): query i sees keys
    spans[i][0] <= j < spans[i][1], clamped to the keys that there are; None: all. A query that sees none gets zeros; what it
    does not see does not reach it, be it NaN. Scores are q . k * scale (>= 0, default hd^-1/2), capped to
    softcap * tanh(s / softcap) where softcap > 0, less slopes[h] |i + Tk - Tq - j| where slopes (fp32 [H]) are given.
    """
    t = q.dtype
    if t is not torch.bfloat16 and t is not torch.float16:
        raise TypeError(f"q must be bfloat16 or float16, got {t}")
    if k.dtype is not t or v.dtype is not t:
        raise TypeError(f"k and v must be {t} like q, got {k.dtype} and {v.dtype}")
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"q must be [B][Tq][H][hd], k and v [B][Tk][Hkv][hd], got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    b, tq, h, hd = q.shape
    tk, hkv = k.shape[1], k.shape[2]
    if k.shape[0] != b or k.shape[3] != hd or hkv < 1 or h < 1 or h % hkv or hd < 8 or hd % 8 or hd > 256:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)}: need equal B and hd (a multiple of 8 up to 256), and H "
                         "a multiple of Hkv")
    strides = _lib.strides3(q), _lib.strides3(k), _lib.strides3(v)
    for s, x in zip(strides, (q, k, v)):
        if x.stride(3) != 1 or s[0] % 8 or s[1] % 8 or s[2] % 8 or x.data_ptr() % 16:
            raise ValueError("q, k and v must have contiguous dims and strides that are multiples of 8, 16-byte aligned, got "
                             f"{x.stride()}")
    scale = hd ** -0.5 if scale is None else float(scale)
    softcap = float(softcap)
    if not 0.0 <= softcap < float("inf") or not 0.0 <= scale < float("inf"):
        raise ValueError(f"scale and softcap must be finite and >= 0, got {scale} and {softcap}")
    index = q.get_device()
    if index < 0 or k.get_device() != index or v.get_device() != index:
        raise ValueError("q, k and v must be on the same GPU")
    if spans is not None:
        if spans.dtype is not torch.int32 or (spans.shape != (b, tq, 2) and spans.shape != (tq, 2)) or spans.get_device() != index:
            raise ValueError(f"spans must be int32 [{b}][{tq}][2] or [{tq}][2] on q's GPU, got {spans.dtype} {tuple(spans.shape)}")
        if spans.dim() == 2 and b > 1:
            spans = spans.expand(b, tq, 2)
        spans = spans.contiguous()
    if slopes is not None and (slopes.dtype is not torch.float32 or slopes.shape != (h,) or not slopes.is_contiguous()
                               or slopes.get_device() != index):
        raise ValueError(f"slopes must be contiguous float32 [{h}] on q's GPU, got {slopes.dtype} {tuple(slopes.shape)}")
    if out is None:
        out = q.new_empty((b, tq, h, hd))
    elif out.dtype is not t or out.shape != q.shape or not out.is_contiguous() or out.get_device() != index or out.data_ptr() % 16:
        raise ValueError(f"out must be contiguous, 16-byte aligned {t} {tuple(q.shape)}, got {out.dtype} {tuple(out.shape)}")
    elif (_lib.overlap(out, k) or _lib.overlap(out, v)
          or _lib.overlap(out, q) and (out.data_ptr() != q.data_ptr() or not q.is_contiguous())):
        raise ValueError("out must not share memory with k or v, nor with q but for being it")
    elif (spans is not None and _lib.overlap(out, spans)) or (slopes is not None and _lib.overlap(out, slopes)):
        raise ValueError("out must not share memory with spans or slopes")
    need = _workspace_bytes(b, tq, tk, h, hd)
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    a = _lib.SpanArgs(_lib.DTYPES[t], q.data_ptr(), _S3(*strides[0]), k.data_ptr(), _S3(*strides[1]), v.data_ptr(),
                      _S3(*strides[2]), None if spans is None else spans.data_ptr(),
                      None if slopes is None else slopes.data_ptr(), b, tq, tk, h, hkv, hd,
                      scale, softcap, out.data_ptr(), None if ws is None else ws.data_ptr(), need)
    _lib.run_on(index, _lib.lib().fa_span_attention, a, "fa_span_attention")
    return out
