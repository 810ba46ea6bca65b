"""lora.add where the choice between its variants goes by the rows: tokens of many requests and prompts past 64 rows, tiles whose adapters
several workgroups deal among them, neighbouring tiles on one XCD, two adapters with one reading of x."""
import pytest
import torch

from flashact_amd import lora
from tests.test_gpu_lora import BF16, F16, F32, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,ytype", [(BF16, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("rows,run", [(65, 1), (65, 3), (129, 16), (257, 5), (600, 1), (1009, 40), (1025, 3), (1601, 293)])
@pytest.mark.parametrize("n,k,rank", [(260, 264, 16), (1030, 136, 8), (72, 2048, 40)])
def test_rows(gpu, dtype, ytype, rows, run, n, k, rank):
    y, x, bank, index, out = _run(gpu, rows, n, k, rank, 11, dtype, ytype, run, seed=rows)
    for _ in range(3):
        assert torch.equal(lora.add(y, x, bank, index), out)
    assert torch.equal(lora.add(y, x, bank, index, out=y), out) and torch.equal(y, out)


@pytest.mark.parametrize("rows,run", [(130, 2), (700, 4), (1100, 37)])
def test_gated_rows(gpu, rows, run):
    _run(gpu, rows, 516, 264, 16, 6, BF16, F32, run, gate=True)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,run", [(100, 1), (100, 5), (1100, 19)])
def test_what_is_not_finite_stays_with_its_request(gpu, dtype, rows, run):
    """Of two adapters whose products are taken together, one is NaN; of a tile's rows, one is."""
    y, x, bank, index, out = _run(gpu, rows, 96, 136, 16, 4, dtype, F32, run)
    for bad in range(4):
        other = {m: t.clone() for m, t in bank.items()}
        other["a"][bad, 3] = float("nan")
        got = lora.add(y, x, other, index)
        assert torch.equal(got[index != bad], out[index != bad]) and bool(got[index == bad].isnan().all())
    row = int((index == 2).nonzero()[0])
    x[row, 7] = float("nan")
    got = lora.add(y, x, bank, index)
    keep = torch.arange(rows, device=gpu) != row
    assert torch.equal(got[keep], out[keep]) and bool(got[row].isnan().all())
