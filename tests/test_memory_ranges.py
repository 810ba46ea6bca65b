"""Which tensors share elements (flashact_amd/_lib.py): against every pair of them."""
import random

import torch

from flashact_amd import _lib


def _places(t):
    i = torch.zeros((), dtype=torch.long)
    for s, n in zip(t.stride(), t.shape):
        i = i[..., None] + s * torch.arange(n)
    return (t.storage_offset() + i).flatten().tolist()


def _view(rng, buf):
    dims = rng.randint(1, 4)
    while True:
        shape = [rng.randint(1, 4) for _ in range(dims)]
        stride = [rng.choice((0, 1, 1, 2, 3, 4, 5, 8, 12, 16, 30)) for _ in range(dims)]
        reach = sum(s * (n - 1) for s, n in zip(stride, shape))
        if reach < buf.numel():
            return torch.as_strided(buf, shape, stride, rng.randint(0, buf.numel() - 1 - reach))


def test_meet_and_doubled_against_every_pair():
    rng, buf, seen = random.Random(0), torch.zeros(200), [0, 0]
    for _ in range(4000):
        a, b = _view(rng, buf), _view(rng, buf)
        if rng.random() < 0.3:  # two views of one layout
            shift = rng.randint(-20, 20)
            at = a.storage_offset() + shift
            if 0 <= at and at + max(_places(a)) - a.storage_offset() < buf.numel():
                b = torch.as_strided(buf, a.shape, a.stride(), at)
        want = bool(set(_places(a)) & set(_places(b)))
        assert _lib.meet(a, b) == _lib.meet(b, a) == want
        seen[want] += 1
        if not _lib.doubled(a):  # it may refuse a layout whose strides are not nested, but never passes one that doubles
            assert len(set(_places(a))) == a.numel()
    assert min(seen) > 500


def test_ordinary_layouts_pass():
    kv = torch.zeros(2, 30, 2, 3, 64)
    assert not _lib.meet(kv[:, :, 0], kv[:, :, 1]) and not _lib.doubled(kv[:, :, 0])
    layers = torch.zeros(3, 4, 2, 16 * 64)  # a sample's keys in rows, its values transposed, side by side
    k, v = layers[:, 1, 0].view(3, 16, 64), layers[:, 1, 1].view(3, 64, 16).transpose(1, 2)
    assert not _lib.meet(k, v) and not _lib.doubled(v) and _lib.meet(k, layers[:, 1, 0].view(3, 64, 16).transpose(1, 2))
    rows = torch.zeros(100, 64)
    assert _lib.meet(rows[:60], rows[59:]) and not _lib.meet(rows[:60], rows[60:]) and not _lib.meet(rows[::2], rows[1::2])
    assert not _lib.meet(rows[:0], rows) and not _lib.doubled(rows[:0])
    assert _lib.doubled(torch.zeros(10).unfold(0, 4, 2)) and _lib.doubled(torch.zeros(1).expand(5))
    assert not _lib.overlap(rows[50:50], rows) and _lib.overlap(rows[50:51], rows) and not _lib.overlap(rows[50:51], rows[51:])
    large = torch.zeros(1).expand(1 << 20, 1 << 10)[:, :0]
    assert not _lib.doubled(large)
