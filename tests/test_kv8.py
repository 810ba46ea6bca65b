"""The 8-bit cache (flashact_amd/kv8.py) on the CPU: shapes, and the requests that its calls and C entries refuse."""
import ctypes

import pytest
import torch

from flashact_amd import _lib, kv8
from tests import kv8_case as C


def test_make_caches():
    caches = kv8.make_caches(3, 2, 70, 4, 96, "cpu")
    assert len(caches) == 3
    for c in caches:
        assert c["k"].shape == (2, 4, 3, 6, 32, 16) and c["v"].shape == (2, 4, 3, 96, 32)
        assert c["ks"].shape == c["vs"].shape == (2, 4, 3) and not c["k"].any() and not c["v"].any()
    assert caches[0]["k"].data_ptr() != caches[1]["k"].data_ptr()
    for bad in ((0, 1, 32, 1, 64), (1, 0, 32, 1, 64), (1, 1, 0, 1, 64), (1, 1, 32, 0, 64), (1, 1, 32, 1, 80)):
        with pytest.raises(ValueError):
            kv8.make_caches(*bad, "cpu")


def test_the_rule_of_scales():
    """The tests' own rule against its bounds: the scale is a power of two, and the largest value uses its last octave."""
    for x in (1.0, 447.9, 448.0, 448.1, 1e-30, 3e38, 5e-42, 1.75 * 2.0 ** 7, 0.0):
        s = C.scale_for(x)
        assert x <= 448 * s and (x > 224 * s or s == 2.0 ** -100)


def _cache():
    return kv8.make_caches(1, 2, 64, 2, 128, "cpu")[0]


def _at(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_calls_refuse():
    c, k = _cache(), torch.randn(2, 3, 2, 128).bfloat16()
    for kw, err, text in ((dict(k=k.double(), v=k.double()), TypeError, "both be"), (dict(k=k[:1]), ValueError, "must be"),
                          (dict(v=k[..., :64]), ValueError, "must be"), (dict(), ValueError, "GPU"),
                          (dict(cache=dict(c, ks=c["ks"][:1])), ValueError, "belong"),
                          (dict(cache=dict(c, k=c["k"].int())), TypeError, "uint8"),
                          (dict(cache=dict(c, v=c["v"][..., :16])), ValueError, "cache v"),
                          (dict(cache={n: t[:0] for n, t in c.items()}), ValueError, "empty"),
                          (dict(cache=dict(c, v=c["v"].transpose(0, 1).contiguous().transpose(0, 1))), ValueError, "contiguous")):
        with pytest.raises(err, match=text):
            kv8.store(**{"cache": c, "k": k, "v": k, "start": _at(0, 0), **kw})
    for kw, err, text in ((dict(k=k), ValueError, "both"), (dict(dtype=torch.float64), TypeError, "dtype"), (dict(), ValueError, "GPU")):
        with pytest.raises(err, match=text):
            kv8.load(**{"cache": c, "lens": _at(0, 0), **kw})
    q = torch.randn(2, 1, 4, 128).bfloat16()
    for kw, err, text in ((dict(q=q.float()), TypeError, "q must"), (dict(q=q[0]), ValueError, "q must"),
                          (dict(q=q[:, :, :3]), ValueError, "multiple of 2"), (dict(softcap=float("inf")), ValueError, "softcap"),
                          (dict(), ValueError, "GPU")):
        with pytest.raises(err, match=text):
            kv8.attend(**{"q": q, "cache": c, "lens": _at(0, 0), **kw})


FAKE = 1 << 20  # aligned dummy addresses: validation must fail before anything is dereferenced


def _rows_args(**kw):
    a = _lib.Kv8RowsArgs()
    for f in ("k", "v", "cache_k", "cache_v", "cache_ks", "cache_vs", "start", "count"):
        setattr(a, f, FAKE)
    a.k_stride = a.v_stride = (ctypes.c_longlong * 4)(256, 256, 128, 1)
    a.batch, a.tokens, a.kv_heads, a.head_dim, a.blocks = 2, 5, 2, 128, 4
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("entry", ["fa_kv8_store", "fa_kv8_load"])
@pytest.mark.parametrize("kw,text", [
    (dict(dtype=1), "dtype"), (dict(batch=0), "batch=0"), (dict(kv_heads=0), "kv_heads=0"), (dict(blocks=0), "blocks=0"),
    (dict(head_dim=80), "head_dim=80"), (dict(tokens=-1), "tokens=-1"), (dict(k=None), "NULL"), (dict(cache_v=None), "NULL"),
    (dict(cache_k=FAKE + 8), "not 16-byte aligned"), (dict(v=FAKE + 1), "not aligned"), (dict(count=FAKE + 2), "4-byte"),
    (dict(start=None, count=None), "is NULL"), (dict(tokens=1 << 29, batch=1 << 10), "too many rows"),
])
def test_row_entries_refuse(entry, kw, text):
    lib = _lib.lib()
    assert getattr(lib, entry)(ctypes.byref(_rows_args(**kw)), None) == 1
    assert text in lib.fa_last_error().decode()


def _attn_args(**kw):
    a = _lib.Kv8AttnArgs()
    for f in ("q", "cache_k", "cache_v", "cache_ks", "cache_vs", "lens", "out", "workspace"):
        setattr(a, f, FAKE)
    a.q_stride = (ctypes.c_longlong * 3)(1024, 1024, 128)
    a.batch, a.tokens, a.heads, a.kv_heads, a.head_dim, a.blocks, a.scale = 2, 1, 8, 2, 128, 400, 0.1
    a.workspace_bytes = 1 << 30
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), "dtype"), (dict(heads=7), "heads=7"), (dict(heads=0), "heads=0"), (dict(head_dim=32), "head_dim=32"),
    (dict(tokens=-1), "tokens=-1"), (dict(tokens=1 << 22), "2^24"), (dict(softcap=-1.0), "softcap"),
    (dict(softcap=float("nan")), "softcap"), (dict(scale=1.0, softcap=1e-39), "fp32 range"), (dict(scale=float("inf")), "scale"), (dict(q=None), "NULL"),
    (dict(out=FAKE + 8), "16-byte"), (dict(lens=FAKE + 2), "4-byte"), (dict(workspace=None), "workspace"),
    (dict(workspace_bytes=100), "workspace"), (dict(q_stride=(ctypes.c_longlong * 3)(1024, 1024, 100)), "q_stride"),
])
def test_attention_entry_refuses(kw, text):
    lib = _lib.lib()
    assert lib.fa_kv8_attention(ctypes.byref(_attn_args(**kw)), None) == 1
    assert text in lib.fa_last_error().decode()


def test_entries_without_work_or_device():
    lib = _lib.lib()
    for f in (lib.fa_kv8_store, lib.fa_kv8_load, lib.fa_kv8_attention):
        assert f(None, None) == 1
    assert lib.fa_kv8_store(ctypes.byref(_rows_args(tokens=0)), None) == 0
    assert lib.fa_kv8_attention(ctypes.byref(_attn_args(tokens=0)), None) == 0
    assert lib.fa_kv8_attention_workspace_bytes(0, 1, 8, 1, 256, 4) == 0
    if not torch.cuda.is_available():
        assert lib.fa_kv8_store(ctypes.byref(_rows_args()), None) == 3
        assert lib.fa_kv8_attention(ctypes.byref(_attn_args()), None) == 3
