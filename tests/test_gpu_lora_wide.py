"""lora.add of up to 64 rows to many columns, where fewer workgroups than a tile has adapters deal these among them."""
import pytest
import torch

from flashact_amd import lora
from tests.test_gpu_lora import BF16, F16, F32, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,run", [(5, 1), (16, 1), (33, 1), (33, 2), (64, 1), (64, 17), (64, 64)])
@pytest.mark.parametrize("n,rank,gate", [(32768, 32, True), (16384, 16, False), (33002, 40, False)])
def test_columns(gpu, dtype, rows, run, n, rank, gate):
    y, x, bank, index, out = _run(gpu, rows, n, 264, rank, 15, dtype, F32, run, gate, seed=rows)
    one = lora.add(y[rows // 2:rows // 2 + 1], x[rows // 2:rows // 2 + 1], bank, index[rows // 2:rows // 2 + 1].clone(), gate="gelu" if gate else None)
    assert torch.equal(one[0], out[rows // 2])  # by itself: one tile of one row, other shares
    if not gate:
        assert torch.equal(lora.add(y, x, bank, index, out=y), out) and torch.equal(y, out)
