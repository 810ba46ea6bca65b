"""paged.append refuses rows that lie in the pool that it writes (the checks come before the devices', so that a CPU tells)."""
import pytest
import torch

from flashact_amd import paged


def _call(k_pool, v_pool, **rows):
    table, start = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    paged.append({"k": k_pool, "v": v_pool}, table, start=start, **rows)


def test_rows_inside_the_pool_are_refused():
    pool = paged.make_pools(1, 6, 1, 64, device="cpu")[0]
    k, v, q = (torch.zeros(2, 3, 1, 64, dtype=torch.bfloat16) for _ in range(3))
    for name in ("k", "v", "q"):
        for which in ("k", "v"):
            for at in (0, 64, pool[which].numel() - 384):
                inside = pool[which].view(-1)[at:at + 384].view(2, 3, 1, 64)
                with pytest.raises(ValueError, match="share memory with the pool"):
                    _call(pool["k"], pool["v"], **{**dict(k=k, v=v, q=q), name: inside})


def test_rows_beside_the_pool_are_not():
    """Neighbours in one allocation, and rows without elements, get as far as the devices' check."""
    n = 6 * 32 * 64
    whole = torch.zeros(2 * n + 3 * 384, dtype=torch.bfloat16)
    rows = [whole[384 + 2 * n:][:384].view(2, 3, 1, 64), whole[:384].view(2, 3, 1, 64), whole[768 + 2 * n:].view(2, 3, 1, 64)]
    k_pool, v_pool = whole[384:384 + n].view(6, 1, 8, 32, 8), whole[384 + n:384 + 2 * n].view(6, 1, 4, 64, 8)
    with pytest.raises(ValueError, match="on one GPU"):
        _call(k_pool, v_pool, k=rows[0], v=rows[1], q=rows[2])
    with pytest.raises(ValueError, match="on one GPU"):
        _call(k_pool, v_pool, k=rows[0], v=rows[1])
    none = k_pool.view(-1)[64:64].view(2, 0, 1, 64)
    with pytest.raises(ValueError, match="on one GPU"):
        _call(k_pool, v_pool, k=none, v=none, q=none)
