"""What the backbone answers, on MI355X: log probabilities of tokens out of logits, with entropy and the best alternatives.

``logprobs`` reads the logits once (C ABI ``fa_token_logprobs``): scoring given tokens, choosing the next one (the first
alternative is the greedy choice), temperatures, vocabularies with tokens ruled out by -inf.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch

from . import _lib

MAX_TOP = 32
_DT = _lib.DTYPES


class LogProbs(NamedTuple):
    logprob: torch.Tensor                 # fp32, the tokens' shape
    entropy: torch.Tensor                 # fp32, the tokens' shape
    top_tokens: Optional[torch.Tensor]    # int32, the tokens' shape x top (None: top = 0)
    top_logprobs: Optional[torch.Tensor]  # fp32, like top_tokens


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(dtype, rows, vocabulary, top) -> int:
    """A function of the sizes alone."""
    return _lib.lib().fa_token_logprobs_workspace_bytes(dtype, rows, vocabulary, top)


@functools.lru_cache(maxsize=1024)
def _logprobs_of(logits, tokens, top):
    """(the struct's type, the rows' stride, whether tokens are 64 bits, rows, vocabulary, the workspace's bytes) of layouts
    (``_lib.layout``), checked: done once for each of them."""
    t = _DT.get(logits[0])
    if t is None:
        raise TypeError(f"logits must be bfloat16, float16 or float32, got {logits[0]}")
    if tokens[0] is not torch.int32 and tokens[0] is not torch.int64:
        raise TypeError(f"tokens must be int32 or int64, got {tokens[0]}")
    dim, shape = len(logits[1]), tokens[1]
    if dim not in (2, 3) or shape != logits[1][:-1] or (dim == 3 and not _lib.contiguous(logits)):
        raise ValueError(f"logits must be [rows][V] or contiguous [B][T][V] and tokens [rows] or [B][T], got {tuple(logits[1])} and "
                         f"{tuple(shape)}")
    rows, vocabulary = shape.numel(), logits[1][-1]
    if vocabulary < 1 or logits[2][-1] != 1 or not _lib.contiguous(tokens):
        raise ValueError(f"logits must have contiguous rows that are not empty and tokens be contiguous, got {tuple(logits[1])} with "
                         f"strides {logits[2]} and {tokens[2]}")
    if rows > 1 << 20 or vocabulary > 1 << 30:
        raise ValueError(f"rows={rows} must be at most 2^20 and the vocabulary of {vocabulary} at most 2^30")
    if not 0 <= top <= min(MAX_TOP, vocabulary):
        raise ValueError(f"top must be in [0, {min(MAX_TOP, vocabulary)}], got {top}")
    return (t, logits[2][0] if dim == 2 else vocabulary, int(tokens[0] is torch.int64), rows, vocabulary,
            _workspace_bytes(t, rows, vocabulary, top) if rows else 0)


def logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0, scale: float = 1.0) -> LogProbs:
    """Log probabilities of `tokens` under softmax(scale * logits), its entropy, and the `top` most probable tokens, on the current
    stream.

    logits [rows][V] (or [B][T][V], contiguous) bf16, fp16 or fp32, dims of V contiguous, rows of any stride and alignment;
    tokens int32 or int64 [rows] (or [B][T]) on the GPU; scale > 0: one over the temperature. Results are fp32, natural
    logarithms. Alternatives come by descending logit, equal ones by ascending token. A logit of -inf rules its token out: log
    probability -inf; where it rules out all of a row, the entropy is 0. A token outside [0, V) has log probability -inf. A row
    with a NaN or +inf has log probabilities and entropy NaN; a NaN is no alternative (token -1 where fewer than `top` are left).
    """
    dtype, stride, wide, rows, vocabulary, need = _logprobs_of(_lib.layout(logits), _lib.layout(tokens), top)
    if not 0.0 < scale < 2e38:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    index = logits.get_device()
    if index < 0 or tokens.get_device() != index:
        raise ValueError(f"logits and tokens must be on the same GPU, got {logits.device} and {tokens.device}")
    logprob = torch.empty_like(tokens, dtype=torch.float32)
    entropy = torch.empty_like(logprob)
    top_logprobs = logprob.new_empty((*tokens.shape, top)) if top else None
    top_tokens = torch.empty_like(top_logprobs, dtype=torch.int32) if top else None
    if rows:
        ws = logprob.new_empty((need + 3) // 4) if need else None
        a = _lib.TokenLogprobsArgs(dtype, logits.data_ptr(), stride, tokens.data_ptr(), wide, scale, rows, vocabulary, top,
                                   logprob.data_ptr(), entropy.data_ptr(), top_tokens.data_ptr() if top else None,
                                   top_logprobs.data_ptr() if top else None, None if ws is None else ws.data_ptr(), need)
        _lib.run_on(index, _lib.lib().fa_token_logprobs, a, "fa_token_logprobs")
    return LogProbs(logprob, entropy, top_tokens, top_logprobs)
