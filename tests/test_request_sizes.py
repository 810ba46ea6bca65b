"""Sizes past those of the C entries are refused in Python, where ctypes would cut them off to 32 bits (tensors without memory)."""
import pytest
import torch

from flashact_amd import lora

META = dict(device="meta")


def _none(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, **META)


@pytest.mark.parametrize("rows,n,k", [(3, 64, 2 ** 24 + 8), (3, 64, 2 ** 32 + 8), (3, 2 ** 24 + 1, 64), (3, 2 ** 32 + 4, 64), (2 ** 32 + 4, 64, 64)])
def test_adapters(rows, n, k):
    bank = {"a": _none(1, k // 8, 8, 8), "b": _none(1, 1, n, 8), "scale": _none(1, dtype=torch.float32)}
    with pytest.raises(ValueError, match="2\\^24"):
        lora.add(_none(rows, n), _none(rows, k), bank, _none(rows, dtype=torch.int32))
