"""Low-rank adapters (flashact_amd/lora.py) on the CPU: packing, and the requests that the call and the C entry refuse."""
import ctypes

import pytest
import torch

from flashact_amd import _lib, lora
from tests import lora_case as C


def test_pack_keeps_the_adapters():
    ads = [(torch.randn(5, 24), torch.randn(10, 5), 2.0), (torch.randn(16, 24), torch.randn(10, 16), -0.25)]
    bank = lora.pack(ads, torch.float16)
    assert bank["a"].shape == (2, 3, 16, 8) and bank["b"].shape == (2, 2, 10, 8) and bank["scale"].tolist() == [2.0, -0.25]
    for (a, b, s), (a2, b2, s2) in zip(ads, lora.unpack(bank)):
        r = a.shape[0]
        assert torch.equal(a2[:r], a.half()) and torch.equal(b2[:, :r], b.half()) and s == s2
        assert not a2[r:].any() and not b2[:, r:].any()
    one = (torch.zeros(4, 16), torch.zeros(6, 4), 1.0)
    for bad in ([], [one, (torch.zeros(4, 24), torch.zeros(6, 4), 1.0)], [one, (torch.zeros(4, 16), torch.zeros(7, 4), 1.0)],
                [(torch.zeros(4, 16), torch.zeros(6, 5), 1.0)], [(torch.zeros(129, 16), torch.zeros(6, 129), 1.0)],
                [(torch.zeros(4, 12), torch.zeros(6, 4), 1.0)], [(torch.full((4, 16), float("inf")), torch.zeros(6, 4), 1.0)],
                [(torch.zeros(0, 16), torch.zeros(6, 0), 1.0)]):
        with pytest.raises(ValueError):
            lora.pack(bad)
    with pytest.raises(TypeError):
        lora.pack([one], torch.float32)


def test_the_definition_against_a_loop():
    gen = torch.Generator().manual_seed(0)
    y, x, bank = C.make(gen, "cpu", 3, 8, 6, 16, torch.bfloat16, 5, torch.float32)
    index = torch.tensor([2, -1, 0, 2, 7], dtype=torch.int32)
    out, bound = C.add(y, x, bank, index)
    for m, i in enumerate(index.tolist()):
        want = y[m].double()
        if 0 <= i < 3:
            a, b, s = lora.unpack(bank)[i]
            want = want + s * (b.double() @ (a.double() @ x[m].double()))
        assert float((out[m] - want).abs().max()) < 1e-12 and bool((bound[m] >= 0).all())


def test_call_refuses():
    y, x, bank = C.make(torch.Generator().manual_seed(1), "cpu", 2, 16, 6, 16, torch.bfloat16, 4, torch.float32)
    index = torch.zeros(4, dtype=torch.int32)
    for kw, err, text in ((dict(x=x.float()), TypeError, "x must"), (dict(x=x.half()), TypeError, "bank"), (dict(y=y.half()), TypeError, "y must"),
                          (dict(x=x[:, :8]), ValueError, "x must"), (dict(y=y[:, :4]), ValueError, "y "), (dict(index=index[:2]), ValueError, "index"),
                          (dict(index=index.long()), ValueError, "int32"), (dict(gate="silu"), ValueError, "gate"),
                          (dict(y=y.t().contiguous().t()), ValueError, "contiguous"), (dict(x=x[0]), ValueError, "x must"),
                          (dict(x=x.repeat(1, 2)[:, ::2]), ValueError, "rows that do not overlap"),
                          (dict(x=x[:1].expand(4, 16)), ValueError, "rows that do not overlap"),
                          (dict(bank=dict(bank, a=bank["a"][:1])), ValueError, "bank"), (dict(bank=dict(bank, b=bank["b"][..., :4])), ValueError, "bank"),
                          (dict(bank=dict(bank, scale=bank["scale"].double())), TypeError, "scale"),
                          (dict(bank=dict(bank, scale=bank["scale"][:1])), ValueError, "bank"),
                          (dict(bank=dict(bank, b=bank["b"].transpose(1, 2).contiguous().transpose(1, 2))), ValueError, "contiguous"),
                          (dict(), ValueError, "GPU")):
        with pytest.raises(err, match=text):
            lora.add(**{"y": y, "x": x, "bank": bank, "index": index, **kw})


FAKE = 1 << 20  # aligned dummy addresses: validation must fail before anything is dereferenced


def _args(**kw):
    a = _lib.LoraArgs()
    for f in ("x", "a", "b", "scale", "index", "y", "out", "workspace"):
        setattr(a, f, FAKE)
    a.x_stride, a.rows, a.n, a.k, a.rank, a.adapters, a.workspace_bytes = 2048, 8, 2560, 2048, 16, 4, 1 << 30
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), "dtype 3"), (dict(y_dtype=2), "y_dtype"), (dict(rows=-1), "rows=-1"), (dict(n=0), "n=0"), (dict(k=12), "k=12"),
    (dict(rank=0), "rank=0"), (dict(rank=12), "rank=12"), (dict(rank=136), "rank=136"), (dict(adapters=0), "adapters=0"),
    (dict(gate=1, n=2561), "even n"), (dict(x=None), "x is NULL"), (dict(b=FAKE + 8), "b is not 16-byte"), (dict(index=FAKE + 2), "index"),
    (dict(y=FAKE + 1), "y is not"), (dict(out=None), "out is NULL"), (dict(x_stride=2044), "x_stride"), (dict(x_stride=2000), "x_stride"),
    (dict(workspace=None), "workspace"), (dict(workspace_bytes=16), "workspace"), (dict(workspace=FAKE + 4), "workspace"),
])
def test_entry_refuses(kw, text):
    lib = _lib.lib()
    assert lib.fa_lora_add(ctypes.byref(_args(**kw)), None) == 1
    assert text in lib.fa_last_error().decode()


def test_entry_without_work_or_device():
    lib = _lib.lib()
    assert lib.fa_lora_add(None, None) == 1
    assert lib.fa_lora_add(ctypes.byref(_args(rows=0)), None) == 0
    assert lib.fa_lora_workspace_bytes(0, 2048, 16) == 0 and lib.fa_lora_workspace_bytes(8, 2048, 16) >= 8 * 16 * 4
    if not torch.cuda.is_available():
        assert lib.fa_lora_add(ctypes.byref(_args()), None) == 3
