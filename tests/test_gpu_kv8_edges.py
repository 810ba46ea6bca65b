"""Edges of the 8-bit cache's attention on the MI355X: caps."""
import pytest
import torch

from flashact_amd import kv8
from tests import kv8_case as C
from tests.test_gpu_kv8 import _filled, _ints

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _put(cache, name, token, codes):
    """Codes [hd] of one token of sample 0, head 0."""
    blk, t = token // kv8.BLOCK, token % kv8.BLOCK
    if name == "k":
        cache["k"][0, 0, blk, :, t] = codes.view(-1, 16)
    else:
        cache["v"][0, 0, blk, :, t] = codes


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("slopes", [False, True])
def test_a_cap_is_each_scores_own(gpu, dtype, slopes):
    """Large scores of other rows, or of keys that a row does not see, do not change a bit of its result."""
    n = 300
    cache, lens = _filled(gpu, 1, n, 1, 128, seed=3), _ints(gpu, n)
    q = torch.randn(1, 4, 4, 128, generator=torch.Generator(device=gpu).manual_seed(3), device=gpu).to(dtype)
    opt = dict(softcap=20.0, slopes=torch.rand(4, device=gpu) * 0.1 if slopes else None)
    ref = kv8.attend(q, cache, lens, **opt)
    q2 = q.clone()
    q2[0, 1] *= 300
    out = kv8.attend(q2, cache, lens, **opt)
    assert torch.equal(out[:, 0], ref[:, 0]) and torch.equal(out[:, 2:], ref[:, 2:])
    _put(cache, "k", n - 1, torch.where(q[0, 3, 0] < 0, 0xFE, 0x7E).to(torch.uint8))  # seen by the last token alone
    assert torch.equal(kv8.attend(q, cache, lens, **opt)[:, :3], ref[:, :3])


@pytest.mark.parametrize("softcap", [1.0, 8.0, 100.0])
def test_caps_next_to_the_two_forms_border(gpu, softcap):
    """Scores on both sides of the border in every block."""
    cache = _filled(gpu, 1, 200, 1, 64, seed=12)
    q = torch.randn(1, 2, 4, 64, device=gpu).half()
    kc, vc = C.rows_of(cache)
    k, v = C.values(kc, cache["ks"]).to(gpu), C.values(vc, cache["vs"]).to(gpu)
    for scale in (0.35 * softcap / 8, 0.05 * softcap):
        C.check(kv8.attend(q, cache, _ints(gpu, 200), scale=scale, softcap=softcap),
                *C.attend(q, k, v, (200,), scale=scale, softcap=softcap))
