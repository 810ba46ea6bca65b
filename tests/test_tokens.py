"""Log probabilities of tokens (flashact_amd/tokens.py) on the CPU: the definition, and the requests that the call and the C entry
refuse."""
import ctypes
import math

import pytest
import torch

from flashact_amd import _lib, tokens
from tests import tokens_case as C


def test_the_definition():
    x = torch.tensor([[0.0, math.log(3.0), -math.inf, 0.0], [-math.inf] * 4])
    ref, _ = C.logprobs(x, torch.tensor([1, 2]), 3)
    assert torch.allclose(ref["logprob"], torch.tensor([math.log(0.6), -math.inf]).double())
    h = -(0.6 * math.log(0.6) + 0.4 * math.log(0.2))
    assert torch.allclose(ref["entropy"], torch.tensor([h, 0.0]).double())
    assert ref["top_tokens"].tolist() == [[1, 0, 3], [0, 1, 2]]
    assert torch.allclose(ref["top_logprobs"][0].exp(), torch.tensor([0.6, 0.2, 0.2]).double())


def test_call_refuses():
    x, t = torch.randn(4, 9), torch.zeros(4, dtype=torch.int64)
    for kw, err, text in ((dict(logits=x.double()), TypeError, "logits"), (dict(tokens=t.short()), TypeError, "tokens"),
                          (dict(logits=x[0]), ValueError, "logits"), (dict(tokens=t[:2]), ValueError, "logits"),
                          (dict(logits=x.t().contiguous().t()), ValueError, "contiguous"), (dict(logits=x[:, :0]), ValueError, "empty"),
                          (dict(logits=x.view(2, 2, 9).transpose(0, 1), tokens=t.view(2, 2)), ValueError, "contiguous"),
                          (dict(top=10), ValueError, "top"), (dict(top=-1), ValueError, "top"),
                          (dict(logits=torch.randn(4, 99), top=33), ValueError, "top"), (dict(scale=0.0), ValueError, "scale"),
                          (dict(scale=float("inf")), ValueError, "scale"), (dict(scale=float("nan")), ValueError, "scale"),
                          (dict(tokens=torch.zeros(8, dtype=torch.int64)[::2]), ValueError, "contiguous"), (dict(), ValueError, "GPU")):
        with pytest.raises(err, match=text):
            tokens.logprobs(**{"logits": x, "tokens": t, **kw})


FAKE = 1 << 20  # aligned dummy addresses: validation must fail before anything is dereferenced


def _args(**kw):
    a = _lib.TokenLogprobsArgs()
    for f in ("logits", "tokens", "logprob", "entropy", "top_tokens", "top_logprobs", "workspace"):
        setattr(a, f, FAKE)
    a.stride, a.scale, a.rows, a.vocabulary, a.top, a.workspace_bytes = 100000, 1.0, 2, 100000, 5, 1 << 30
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=1), "dtype 1"), (dict(rows=-1), "rows=-1"), (dict(vocabulary=0), "vocabulary=0"), (dict(vocabulary=(1 << 30) + 1), "vocabulary"),
    (dict(top=33), "top=33"), (dict(top=-1), "top=-1"), (dict(top=9, vocabulary=8), "top=9"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=3e38), "scale"), (dict(logits=None), "logits is NULL"), (dict(logits=FAKE + 1), "logits"),
    (dict(tokens=FAKE + 4, wide_tokens=1), "tokens is not 8-byte"), (dict(top_tokens=None), "top_tokens"), (dict(entropy=FAKE + 2), "entropy"),
    (dict(workspace=None), "workspace"), (dict(workspace_bytes=64), "workspace"), (dict(dtype=3, logits=FAKE + 2), "logits is not 4-byte"),
])
def test_entry_refuses(kw, text):
    lib = _lib.lib()
    assert lib.fa_token_logprobs(ctypes.byref(_args(**kw)), None) == 1
    assert text in lib.fa_last_error().decode()


def test_entry_without_work_or_device():
    lib = _lib.lib()
    assert lib.fa_token_logprobs(None, None) == 1
    assert lib.fa_token_logprobs(ctypes.byref(_args(rows=0)), None) == 0
    assert lib.fa_token_logprobs_workspace_bytes(0, 0, 100, 5) == 0 and lib.fa_token_logprobs_workspace_bytes(0, 2048, 100000, 5) == 0
    assert lib.fa_token_logprobs_workspace_bytes(0, 1, 100000, 5) > 0
    if not torch.cuda.is_available():
        assert lib.fa_token_logprobs(ctypes.byref(_args()), None) == 3
