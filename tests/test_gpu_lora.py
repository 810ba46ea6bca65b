"""Low-rank adapters beside a shared projection on the MI355X, against 64 bits (bounds: lora_case.add)."""
import pytest
import torch

from flashact_amd import lora, w4
from tests import lora_case as C
from tests.kv8_case import check

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _index(gpu, rows, adapters, run=1):
    """Requests of `run` rows: the adapters in turn, then none, then a number that is no adapter's."""
    i = torch.arange(rows, device=gpu) // run % (adapters + 2)
    return torch.where(i == adapters, -1, torch.where(i > adapters, 1 << 30, i)).to(torch.int32)


def _run(gpu, rows, n, k, rank, adapters, dtype, ytype, run=1, gate=False, seed=0):
    y, x, bank = C.make(torch.Generator(device=gpu).manual_seed(seed), gpu, adapters, rank, n, k, dtype, rows, ytype)
    index = _index(gpu, rows, adapters, run)
    out = lora.add(y, x, bank, index, gate="gelu" if gate else None)
    assert out.dtype is (dtype if gate else ytype) and out.shape == (rows, n // 2 if gate else n)
    check(out, *C.add(y, x, bank, index, gate))
    if not gate:
        bare = (index < 0) | (index >= adapters)
        assert torch.equal(out[bare], y[bare])
    return y, x, bank, index, out


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("ytype", [None, F32])
@pytest.mark.parametrize("rows", [1, 2, 15, 17, 64, 300])
@pytest.mark.parametrize("n,k,rank,adapters", [(256, 512, 16, 3), (70, 72, 8, 1), (131, 1032, 24, 17), (1030, 2048, 64, 2), (16, 8, 128, 5)])
def test_add(gpu, dtype, ytype, rows, n, k, rank, adapters):
    _run(gpu, rows, n, k, rank, adapters, dtype, ytype or dtype)
    _run(gpu, rows, n, k, rank, adapters, dtype, ytype or dtype, run=7, seed=1)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("ytype", [None, F32])
@pytest.mark.parametrize("rows,n,k,rank", [(1, 512, 256, 16), (33, 70, 64, 8), (300, 1024, 128, 40)])
def test_gate(gpu, dtype, ytype, rows, n, k, rank):
    _run(gpu, rows, n, k, rank, 3, dtype, ytype or dtype, run=2, gate=True)


@pytest.mark.parametrize("rows,run", [(16, 1), (1500, 211), (700, 1)])
def test_long_sums(gpu, rows, run):
    """K split over workgroups; many rows of one adapter, and every row another one's."""
    _run(gpu, rows, 384, 16384, 16, 9, BF16, F32, run)


def test_outliers_next_to_small_values(gpu):
    """fp16: h far outside of the type's range, next to rows whose h is tiny."""
    y, x, bank = C.make(torch.Generator(device=gpu).manual_seed(3), gpu, 2, 16, 64, 256, F16, 6, F32)
    x[0] *= 6000
    x[1] *= 1e-4
    bank["scale"][0], bank["scale"][1] = 3e4, 1e-12
    y *= 1e-6
    index = torch.tensor([0, 0, 1, 0, 1, -1], dtype=torch.int32, device=gpu)
    check(lora.add(y, x, bank, index), *C.add(y, x, bank, index))
    x[2] = 0
    check(lora.add(y, x, bank, index), *C.add(y, x, bank, index))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows", [5, 40, 300])
def test_a_request_reaches_its_own_rows_only(gpu, dtype, rows):
    """Infinities and NaN in one row's x, and in one adapter, change nothing elsewhere."""
    y, x, bank, index, out = _run(gpu, rows, 96, 136, 16, 3, dtype, F32)
    x2 = x.clone()
    x2[0, 5], x2[4, 7] = float("nan"), float("inf")
    got = lora.add(y, x2, bank, index)
    keep = torch.ones(rows, dtype=torch.bool, device=gpu)
    keep[0] = keep[4] = False
    assert torch.equal(got[keep], out[keep]) and bool(got[0].isnan().all())
    bad = {n: t.clone() for n, t in bank.items()}
    bad["a"][1, 3] = float("nan")
    got = lora.add(y, x, bad, index)
    assert torch.equal(got[index != 1], out[index != 1]) and bool(got[index == 1].isnan().all())
    bad = {n: t.clone() for n, t in bank.items()}
    bad["b"][2, 0, 50:] = float("inf")
    got = lora.add(y, x, bad, index)
    assert torch.equal(got[index != 2], out[index != 2]) and torch.equal(got[:, :50], out[:, :50])


def test_strided_rows_in_place_and_nothing(gpu):
    gen = torch.Generator(device=gpu).manual_seed(7)
    y, x, bank = C.make(gen, gpu, 2, 8, 100, 64, BF16, 9, BF16)
    index = _index(gpu, 9, 2)
    ref = lora.add(y, x, bank, index)
    wide = torch.full((9, 200), float("nan"), device=gpu, dtype=BF16)
    wide[:, 64:128] = x
    assert torch.equal(lora.add(y, wide[:, 64:128], bank, index), ref)
    odd = torch.empty(901, device=gpu, dtype=BF16)[1:].view(9, 100)  # y and out 2-byte aligned
    odd.copy_(y)
    assert torch.equal(lora.add(odd, x, bank, index), ref)
    assert lora.add(odd, x, bank, index, out=odd) is odd and torch.equal(odd, ref)
    assert lora.add(y[:0], x[:0], bank, index[:0]).shape == (0, 100)
    none = torch.full((9,), -1, dtype=torch.int32, device=gpu)
    assert torch.equal(lora.add(y, x, bank, none), y)
    for _ in range(5):
        assert torch.equal(lora.add(y, x, bank, index), ref)
    for out in (x.view(-1)[:0], y[:, :50], torch.empty(9, 100, device=gpu)):
        with pytest.raises(ValueError):
            lora.add(y, x, bank, index, out=out)
    both = torch.randn(18, 100, device=gpu).bfloat16()
    with pytest.raises(ValueError, match="share"):
        lora.add(both[:9], x, bank, index, out=both[4:13])
    with pytest.raises(ValueError, match="share"):
        lora.add(both[:9], x, bank, index, gate="gelu", out=both.view(-1)[:450].view(9, 50))


@pytest.mark.parametrize("rows", [4, 20])
def test_beside_a_projection_in_4_bits(gpu, rows):
    """The gated projection of the MLP as a user composes it: the shared product in fp32, the adapters, the gate."""
    gen = torch.Generator(device=gpu).manual_seed(rows)
    w = w4.quantize(torch.randn(512, 256, generator=gen, device=gpu) * 0.05)
    _, x, bank = C.make(gen, gpu, 3, 16, 512, 256, BF16, rows, F32)
    index = _index(gpu, rows, 3)
    y = w4.linear(x, w, out_dtype=F32)
    check(lora.add(y, x, bank, index, gate="gelu"), *C.add(y, x, bank, index, True))
    none = torch.full_like(index, -1)
    shared, own = lora.add(y, x, bank, none, gate="gelu"), w4.linear(x, w, gate="gelu")
    assert torch.equal(shared, own)  # the same sums and gate
