"""Sizes past those of the C entries are refused in Python, where ctypes would cut them off to 32 bits (tensors without memory)."""
import pytest
import torch

from flashact_amd import lora, paged, tokens

META = dict(device="meta")


def _none(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, **META)


@pytest.mark.parametrize("v", [2 ** 32 + 5, 2 ** 31, 2 ** 30 + 1])
def test_vocabularies(v):
    with pytest.raises(ValueError, match="2\\^30"):
        tokens.logprobs(_none(1, v), _none(1, dtype=torch.int64))


def test_rows_of_tokens():
    with pytest.raises(ValueError, match="2\\^20"):
        tokens.logprobs(_none(1, 8).expand(2 ** 32 + 2, 8), _none(2 ** 32 + 2, dtype=torch.int32))


@pytest.mark.parametrize("rows,n,k", [(3, 64, 2 ** 24 + 8), (3, 64, 2 ** 32 + 8), (3, 2 ** 24 + 1, 64), (3, 2 ** 32 + 4, 64), (2 ** 32 + 4, 64, 64)])
def test_adapters(rows, n, k):
    bank = {"a": _none(1, k // 8, 8, 8), "b": _none(1, 1, n, 8), "scale": _none(1, dtype=torch.float32)}
    with pytest.raises(ValueError, match="2\\^24"):
        lora.add(_none(rows, n), _none(rows, k), bank, _none(rows, dtype=torch.int32))


def test_pages():
    big = 2 ** 32 + 3
    pool = {"k": _none(4, 1, 8, 32, 8), "v": _none(4, 1, 4, 64, 8)}
    table, at = _none(1, 9, dtype=torch.int32), _none(1, dtype=torch.int32)
    row = _none(1, 1, 1, 64)
    long, wide = row.expand(1, big, 1, 64), _none(1, big, dtype=torch.int32)
    for call in (lambda: paged.append(pool, table, long, long, at), lambda: paged.append(pool, wide, row, row, at),
                 lambda: paged.append(pool, table, row, row, at, q=row.expand(1, 1, big, 64)), lambda: paged.load(pool, table, at, k=long, v=long),
                 lambda: paged.load(pool, wide, at, k=row, v=row), lambda: paged.attend(long, pool, table, at),
                 lambda: paged.attend(row, pool, wide, at), lambda: paged.attend(row.expand(1, 1, big, 64), pool, table, at)):
        with pytest.raises(ValueError, match="2\\^31"):
            call()
    many = {n: t[:1].expand(2 ** 31, *t.shape[1:]) for n, t in pool.items()}
    with pytest.raises(ValueError, match="contiguous"):
        paged.attend(row, many, table, at)
