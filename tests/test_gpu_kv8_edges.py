"""Edges of the 8-bit cache's attention on the MI355X: caps, weights far below the largest."""
import math

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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,length", [(1, 131072), (200, 32768)])
def test_many_keys_of_small_weight_count(gpu, dtype, tokens, length):
    """One key outweighs each of the others by e^18, 2^26: together they are 2^-11 to 2^-9 of the sum, and hold all of its value.

    Rounded: the weights (2^-12), the result, and, 2^-12 in all, the score of 18 log2(e) (2^-19) and the sums, of at most 2^10 terms
    a lane (2^-14).
    """
    cache = kv8.make_caches(1, 1, length, 1, 64, gpu)[0]
    cache["v"].fill_(0x38)  # 1
    _put(cache, "k", 5, torch.full((64,), 0x41, dtype=torch.uint8, device=gpu))  # 2.25: 64 x 2.25 / 8 = 18
    _put(cache, "v", 5, torch.zeros(64, dtype=torch.uint8, device=gpu))
    q = torch.ones(1, tokens, 8, 64, device=gpu, dtype=dtype)
    out = kv8.attend(q, cache, _ints(gpu, length), causal=False).double()
    others = (length - 1) * math.exp(-18.0)
    want = others / (1 + others)
    assert bool(((out - want).abs() <= want * (torch.finfo(dtype).eps / 2 + 2.0 ** -11)).all()), (out.min().item(), out.max().item(), want)


def test_scores_and_scales_of_any_size(gpu):
    """Scores of millions, whose differences are whole numbers, and values near the largest of fp32."""
    cache, lens = _filled(gpu, 1, 400, 1, 64, seed=8), _ints(gpu, 400)
    cache["vs"].fill_(2.0 ** 118)
    kc, vc = C.rows_of(cache)
    q = torch.randn(1, 1, 4, 64, device=gpu).bfloat16()
    k, v = C.values(kc, cache["ks"]).to(gpu), C.values(vc, cache["vs"]).to(gpu)
    out = kv8.attend(q, cache, lens)
    C.check(out, *C.attend(q, k, v, (400,)))
    # powers of two times whole keys: products and scores are exact, however large
    cache["ks"].fill_(1.0)
    q = torch.zeros(1, 3, 4, 64, device=gpu, dtype=torch.bfloat16)
    q[0, :, :, 0] = torch.tensor([2.0 ** 12, 2.0 ** 14, 2.0 ** 20], device=gpu)[:, None]
    cache["vs"].fill_(1.0)
    k, v = C.values(kc, cache["ks"]).to(gpu), C.values(vc, cache["vs"]).to(gpu)
    out = kv8.attend(q, cache, lens, scale=1.0, causal=False)
    top = k[0, 0, :400, 0].amax()
    best = v[0, 0, :400][k[0, 0, :400, 0] == top].mean(0)  # neighbouring keys differ by far more than the softmax's range
    assert bool(((out.double() - best).abs() <= 2.0 ** -8 * best.abs() + 2.0 ** -9).all())
