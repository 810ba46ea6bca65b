"""lora.add where K is split over workgroups, whose sums the way back adds: every rank's kernel, both types, two to four splits."""
import pytest
import torch

from flashact_amd import lora
from tests.test_gpu_lora import BF16, F16, F32, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rank,k,splits", [(16, 16384, 2), (16, 24584, 3), (8, 32776, 4), (24, 16384, 2), (32, 24576, 3), (32, 32776, 4),
                                           (40, 8200, 2), (40, 16384, 4), (64, 12288, 3), (72, 4096, 2), (72, 6152, 3), (128, 4104, 2),
                                           (128, 16384, 4), (104, 32776, 4)])
@pytest.mark.parametrize("rows,run,ytype,gate", [(5, 1, F32, False), (40, 3, None, False), (300, 70, F32, True)])
def test_splits(gpu, dtype, rank, k, splits, rows, run, ytype, gate):
    assert lora._workspace_bytes(rows, k, rank) == splits * rows * rank * 4
    y, x, bank, index, out = _run(gpu, rows, 132, k, rank, 5, dtype, ytype or dtype, run, gate, seed=rank)
    for _ in range(3):
        assert torch.equal(lora.add(y, x, bank, index, gate="gelu" if gate else None), out)
