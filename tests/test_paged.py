"""The paged cache (flashact_amd/paged.py) on the CPU: shapes, and the requests that its calls and C entries refuse."""
import ctypes

import pytest
import torch

from flashact_amd import _lib, paged
from tests import paged_case as C


def test_make_pools_and_frequencies():
    pools = paged.make_pools(3, 7, 2, 96, torch.float16, "cpu")
    assert len(pools) == 3
    for p in pools:
        assert p["k"].shape == (7, 2, 12, 32, 8) and p["v"].shape == (7, 2, 4, 96, 8) and p["k"].dtype is torch.float16
        assert not p["k"].any() and not p["v"].any()
    assert pools[0]["k"].data_ptr() != pools[1]["k"].data_ptr()
    for bad in ((0, 1, 1, 64), (1, 0, 1, 64), (1, 1, 0, 64), (1, 1, 1, 80)):
        with pytest.raises(ValueError):
            paged.make_pools(*bad, device="cpu")
    with pytest.raises(TypeError):
        paged.make_pools(1, 1, dtype=torch.float32, device="cpu")
    f = paged.frequencies(64, 1000.0, "cpu")
    assert f.dtype is torch.float64 and f.shape == (32,) and f[0] == 1 and abs(f[31].item() - 1000.0 ** (-62 / 64)) < 1e-15
    for bad in ((0, 10.0), (24, 10.0), (64, 0.0), (64, float("inf"))):
        with pytest.raises(ValueError):
            paged.frequencies(*bad, "cpu")


def test_the_definition_turns_as_the_table_of_the_denoise_loop():
    """The tests' rotation against pi05.rope_table's cosines and sines."""
    from flashact_amd import pi05
    cos, sin = pi05.rope_table(900, 5)
    x = torch.randn(5, 1, 256)
    y, _ = C.turned(x, 900 + torch.arange(5), paged.frequencies(256, device="cpu"), False)
    lo, hi = x[..., :128].double(), x[..., 128:].double()
    c, s = cos.cpu().double()[:, None], sin.cpu().double()[:, None]
    want = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
    assert float((y - want).abs().max()) < 1e-3  # that table's angles are fp32: 900 2^-24 and up
    z, _ = C.turned(torch.stack([x[..., :128], x[..., 128:]], -1).flatten(2), 900 + torch.arange(5),
                    paged.frequencies(256, device="cpu"), True)
    assert torch.equal(y, z)


def _pool():
    return paged.make_pools(1, 6, 2, 128, device="cpu")[0], torch.zeros(2, 3, dtype=torch.int32)


def _at(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_calls_refuse():
    p, table = _pool()
    k = torch.randn(2, 3, 2, 128).bfloat16()
    q = torch.randn(2, 3, 4, 128).bfloat16()
    pools = ((dict(pool=dict(p, k=p["k"][:3])), ValueError, "belong"), (dict(pool=dict(p, k=p["k"].half())), TypeError, "both be"),
             (dict(pool=dict(p, v=p["v"][:, :, :, :64])), ValueError, "belong"), (dict(pool=dict(p, v=p["v"][..., :4])), ValueError, "pool v"),
             (dict(pool={n: t[:0] for n, t in p.items()}), ValueError, "empty"),
             (dict(pool=dict(p, k=p["k"].transpose(0, 1).contiguous().transpose(0, 1))), ValueError, "contiguous"),
             (dict(table=table.long()), ValueError, "table"), (dict(table=table[0]), ValueError, "table"),
             (dict(table=table[:, :0]), ValueError, "table"), (dict(table=torch.zeros(3, 2, dtype=torch.int32).t()), ValueError, "table"),
             (dict(table=table[:1].expand(2, 3)), ValueError, "overlap"), (dict(), ValueError, "GPU"))
    for kw, err, text in pools + ((dict(k=k.float(), v=k.float()), TypeError, "like the pool"), (dict(k=k[:1]), ValueError, "must be"),
                                  (dict(v=k[..., :64]), ValueError, "must be")):
        with pytest.raises(err, match=text):
            paged.append(**{"pool": p, "table": table, "k": k, "v": k, "start": _at(0, 0), **kw})
    for kw, err, text in pools + ((dict(k=k), ValueError, "both"),):
        with pytest.raises(err, match=text):
            paged.load(**{"pool": p, "table": table, "lens": _at(0, 0), **kw})
    for kw, err, text in pools + ((dict(q=q.float()), TypeError, "q must"), (dict(q=q[0]), ValueError, "q must"),
                                  (dict(q=q[:, :, :3]), ValueError, "multiple of 2"), (dict(softcap=float("inf")), ValueError, "softcap"),
                                  (dict(q=q.transpose(2, 3).contiguous().transpose(2, 3)), ValueError, "strides")):
        with pytest.raises(err, match=text):
            paged.attend(**{"q": q, "pool": p, "table": table, "lens": _at(0, 0), **kw})


FAKE = 1 << 20  # aligned dummy addresses: validation must fail before anything is dereferenced


def _rows_args(**kw):
    a = _lib.PagedRowsArgs()
    for f in ("q", "q_out", "k", "v", "pool_k", "pool_v", "table", "start", "count", "freqs"):
        setattr(a, f, FAKE)
    a.k_stride = a.v_stride = (ctypes.c_longlong * 4)(256, 256, 128, 1)
    a.q_stride = (ctypes.c_longlong * 3)(512, 512, 128)
    a.batch, a.tokens, a.heads, a.kv_heads, a.head_dim, a.pages, a.table_pages, a.table_stride, a.rotary = 2, 5, 4, 2, 128, 9, 4, 4, 128
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("entry", ["fa_paged_append", "fa_paged_load"])
@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), "dtype"), (dict(batch=0), "batch=0"), (dict(kv_heads=0), "kv_heads=0"), (dict(pages=0), "pages=0"),
    (dict(table_pages=0), "table_pages=0"), (dict(pages=1 << 30, kv_heads=8), "pages="), (dict(head_dim=80), "head_dim=80"),
    (dict(tokens=-1), "tokens=-1"), (dict(k=None), "NULL"), (dict(pool_v=None), "NULL"), (dict(table=None), "NULL"),
    (dict(pool_k=FAKE + 8), "not 16-byte aligned"), (dict(v=FAKE + 1), "aligned"), (dict(count=FAKE + 2), "4-byte"),
    (dict(table=FAKE + 2), "4-byte"), (dict(table_stride=3), "table_stride=3"), (dict(start=None, count=None), "is NULL"),
    (dict(tokens=1 << 29, batch=1 << 10), "too many rows"),
])
def test_row_entries_refuse(entry, kw, text):
    lib = _lib.lib()
    assert getattr(lib, entry)(ctypes.byref(_rows_args(**kw)), None) == 1
    assert text in lib.fa_last_error().decode()


@pytest.mark.parametrize("kw,text", [
    (dict(k=FAKE + 8), "aligned"), (dict(k_stride=(ctypes.c_longlong * 4)(256, 100, 128, 1)), "multiples of 8"),
    (dict(v_stride=(ctypes.c_longlong * 4)(256, 256, 128, 2)), "contiguous"), (dict(rotary=24), "rotary=24"),
    (dict(rotary=144), "rotary=144"), (dict(rotary=-16), "rotary=-16"), (dict(freqs=None), "freqs"), (dict(freqs=FAKE + 4), "freqs"),
    (dict(q_out=None), "q_out"), (dict(q=FAKE + 8), "q_out"), (dict(heads=0), "heads=0"),
    (dict(q_stride=(ctypes.c_longlong * 3)(512, 512, 100)), "multiples of 8"),
])
def test_append_entry_refuses(kw, text):
    lib = _lib.lib()
    assert lib.fa_paged_append(ctypes.byref(_rows_args(**kw)), None) == 1
    assert text in lib.fa_last_error().decode()


def _attn_args(**kw):
    a = _lib.PagedAttnArgs()
    for f in ("q", "pool_k", "pool_v", "table", "lens", "out", "workspace"):
        setattr(a, f, FAKE)
    a.q_stride = (ctypes.c_longlong * 3)(1024, 1024, 128)
    a.batch, a.tokens, a.heads, a.kv_heads, a.head_dim, a.scale = 2, 1, 8, 2, 128, 0.1
    a.pages, a.table_pages, a.table_stride, a.workspace_bytes = 900, 400, 400, 1 << 30
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), "dtype"), (dict(heads=7), "heads=7"), (dict(heads=0), "heads=0"), (dict(head_dim=32), "head_dim=32"),
    (dict(tokens=-1), "tokens=-1"), (dict(tokens=1 << 22), "2^24"), (dict(softcap=-1.0), "softcap"), (dict(pages=0), "pages=0"),
    (dict(table=None), "NULL"), (dict(table_stride=9), "table_stride"), (dict(softcap=float("nan")), "softcap"),
    (dict(scale=1.0, softcap=1e-39), "fp32 range"), (dict(scale=float("inf")), "scale"), (dict(q=None), "NULL"),
    (dict(out=FAKE + 8), "16-byte"), (dict(lens=FAKE + 2), "4-byte"), (dict(workspace=None), "workspace"),
    (dict(workspace_bytes=100), "workspace"), (dict(q_stride=(ctypes.c_longlong * 3)(1024, 1024, 100)), "q_stride"),
])
def test_attention_entry_refuses(kw, text):
    lib = _lib.lib()
    assert lib.fa_paged_attention(ctypes.byref(_attn_args(**kw)), None) == 1
    assert text in lib.fa_last_error().decode()


def test_entries_without_work_or_device():
    lib = _lib.lib()
    for f in (lib.fa_paged_append, lib.fa_paged_load, lib.fa_paged_attention):
        assert f(None, None) == 1
    assert lib.fa_paged_append(ctypes.byref(_rows_args(tokens=0)), None) == 0
    assert lib.fa_paged_load(ctypes.byref(_rows_args(tokens=0)), None) == 0
    assert lib.fa_paged_attention(ctypes.byref(_attn_args(tokens=0)), None) == 0
    assert lib.fa_paged_attention_workspace_bytes(0, 1, 8, 1, 256, 4) == 0
    if not torch.cuda.is_available():
        assert lib.fa_paged_append(ctypes.byref(_rows_args()), None) == 3
        assert lib.fa_paged_load(ctypes.byref(_rows_args()), None) == 3
        assert lib.fa_paged_attention(ctypes.byref(_attn_args()), None) == 3
