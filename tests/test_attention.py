"""Attention over spans of keys (flashact_amd/attention.py) on the CPU: the spans, and what the call and its C entry refuse."""
import ctypes

import pytest
import torch

from flashact_amd import _lib, attention


def test_prefix_spans():
    t = lambda *v: torch.tensor(v)  # noqa: E731
    s = attention.prefix_spans(t(3, 0, 4), t(2, 0, 9), 9)
    assert s.dtype == torch.int32
    assert s.tolist() == [[0, 2], [0, 2], [0, 3], [3, 7], [3, 7], [3, 7], [3, 7], [0, 0], [0, 0]]
    assert attention.prefix_spans(t(3, 4), t(0, 4), 5).tolist() == [[0, 1], [0, 2], [0, 3], [3, 5], [3, 5]]  # cut off
    assert attention.prefix_spans(t(5)[:0], t(5)[:0], 2).tolist() == [[0, 0], [0, 0]]
    assert attention.prefix_spans(t(-2, 2), t(-1, 0), 3).tolist() == [[0, 1], [0, 2], [0, 0]]
    assert attention.prefix_spans(t(2), t(0), 0).shape == (0, 2)
    for bad in ((t(1.5), t(1), 3), (t(1), t(1.0), 3), (t(1, 2), t(1), 3), (t([1]), t([1]), 3), (t(1), t(1), -1)):
        with pytest.raises(ValueError):
            attention.prefix_spans(*bad)


def test_prefix_spans_against_every_pair():
    g = torch.Generator().manual_seed(0)
    for _ in range(30):
        n = int(torch.randint(1, 5, (1,), generator=g))
        lengths, prefix = torch.randint(0, 7, (n,), generator=g), torch.randint(0, 9, (n,), generator=g)
        total = int(lengths.sum()) + int(torch.randint(0, 4, (1,), generator=g))
        s = attention.prefix_spans(lengths, prefix, total)
        doc = torch.repeat_interleave(torch.arange(n), lengths).tolist() + [-1] * total
        at = [i for x in lengths.tolist() for i in range(x)] + [0] * total
        for i in range(total):
            for j in range(total):
                same = doc[i] >= 0 and doc[i] == doc[j]
                sees = same and (at[j] <= at[i] or at[j] < int(prefix[doc[i]]))
                assert sees == (int(s[i, 0]) <= j < int(s[i, 1]))


def test_attend_refuses():
    q, k = torch.randn(2, 8, 4, 64).bfloat16(), torch.randn(2, 8, 2, 64).bfloat16()
    for kw, err, text in ((dict(q=q.float()), TypeError, "q must be"), (dict(k=k.half()), TypeError, "like q"),
                          (dict(q=q[0]), ValueError, "must be"), (dict(v=k[:, :7]), ValueError, "must be"),
                          (dict(k=k[:1], v=k[:1]), ValueError, "equal B"), (dict(q=q[..., :60]), ValueError, "equal B"),
                          (dict(q=q[:, :, :3]), ValueError, "multiple of Hkv"),
                          (dict(q=q[..., :12], k=k[..., :12], v=k[..., :12]), ValueError, "multiple of 8"),
                          (dict(q=q.transpose(1, 3).contiguous().transpose(1, 3)), ValueError, "contiguous dims"),
                          (dict(softcap=float("nan")), ValueError, "softcap"), (dict(scale=-1.0), ValueError, "scale"),
                          (dict(), ValueError, "same GPU")):
        with pytest.raises(err, match=text):
            attention.attend(**{"q": q, "k": k, "v": k, **kw})
    wide = torch.randn(1, 2, 1, 264).bfloat16()
    with pytest.raises(ValueError, match="up to 256"):
        attention.attend(wide, wide, wide)


FAKE = 1 << 20  # aligned dummy addresses: validation must fail before anything is dereferenced


def _args(**kw):
    a = _lib.SpanArgs()
    a.q = a.k = a.v = a.out = FAKE
    a.q_stride = a.k_stride = a.v_stride = (ctypes.c_longlong * 3)(8192, 1024, 128)
    a.batch, a.queries, a.keys, a.heads, a.kv_heads, a.head_dim, a.scale = 2, 8, 8, 4, 2, 128, 0.1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=3), 1, "dtype"), (dict(batch=-1), 1, "batch=-1"), (dict(keys=-1), 1, "keys=-1"),
    (dict(heads=5), 1, "heads=5"), (dict(kv_heads=0), 1, "kv_heads=0"), (dict(head_dim=260), 1, "head_dim=260"),
    (dict(head_dim=12), 1, "head_dim=12"), (dict(softcap=-1.0), 1, "softcap"), (dict(scale=float("nan")), 1, "scale"),
    (dict(scale=-1.0), 1, "scale"), (dict(scale=1.0, softcap=1e-39), 1, "fp32 range"), (dict(v=None), 1, "NULL"), (dict(k=FAKE + 8), 1, "16-byte"),
    (dict(spans=FAKE + 2), 1, "4-byte"), (dict(q_stride=(ctypes.c_longlong * 3)(0, 4, 8)), 1, "multiples of 8"),
    (dict(k_stride=(ctypes.c_longlong * 3)(0, 1 << 24, 8)), 2, "2^23"),
    (dict(v_stride=(ctypes.c_longlong * 3)(0, -8, 8)), 2, "2^23"),
])
def test_c_entry_refuses(kw, code, text):
    lib = _lib.lib()
    assert lib.fa_span_attention(ctypes.byref(_args(**kw)), None) == code
    assert text in lib.fa_last_error().decode()


def test_c_entry_without_work_or_device():
    lib = _lib.lib()
    assert lib.fa_span_attention(None, None) == 1
    assert lib.fa_span_attention(ctypes.byref(_args(queries=0)), None) == 0
    assert lib.fa_span_attention(ctypes.byref(_args(batch=0)), None) == 0
    if not torch.cuda.is_available():
        assert lib.fa_span_attention(ctypes.byref(_args()), None) == 3


def test_c_entry_workspace():
    """Few queries over many keys have a use for one, few keys or many queries none; one that is too small is refused."""
    lib = _lib.lib()
    need = lib.fa_span_attention_workspace_bytes
    assert need(1, 1, 100000, 8, 128) > 0 and need(1, 64, 4096, 8, 256) > 0
    assert need(1, 1, 100, 8, 128) == need(1, 8192, 8192, 16, 128) == need(0, 1, 1, 1, 1) == need(1, 0, 9, 1, 8) == 0
    assert need(1, 1, 1 << 30, 1, 256) <= 80 << 20  # bounded: no more than 1024 parts of 64 rows
    n = need(2, 8, 9000, 4, 128)
    a = _args(keys=9000, workspace=FAKE, workspace_bytes=n - 1)
    assert lib.fa_span_attention(ctypes.byref(a), None) == 1 and "workspace" in lib.fa_last_error().decode()
    a = _args(keys=9000, workspace=FAKE + 8, workspace_bytes=n)
    assert lib.fa_span_attention(ctypes.byref(a), None) == 1 and "16-byte" in lib.fa_last_error().decode()
