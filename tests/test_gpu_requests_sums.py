"""Adapters on the way back into the fp32 residual stream of packed prompts: their sums keep fp32."""
import pytest
import torch

from flashact_amd import kv8, paged, prefill
from tests.test_gpu_backbone import NL, _ints, _weights
from tests.test_gpu_requests import _banks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["wo", "wdn"])
@pytest.mark.parametrize("pages", [True, False])
def test_twice_the_scale_adds_twice_as_much(gpu, name, pages):
    """An adapter of the last layer alone, whose sum goes into the result as it is (wo: the MLP's way back is zero).

    Twice the scale, a power of two, doubles the adapter's sum exactly; the sum with y and the residual is rounded to fp32 once or
    twice, 2^-24 of the result each, in each of the three calls: below 2^-21 of the largest of their elements.
    """
    _, packed, _, ln = _weights(gpu, seed=5)
    packed = dict(packed)
    if name == "wo":
        packed["wdn"] = packed["wdn"].clone()
        packed["wdn"][-1] = 0
    banks = [{}] * (NL - 1) + [{name: _banks(gpu, 6, (name,))[-1][name]}]
    twice = [{}] * (NL - 1) + [{name: dict(banks[-1][name], scale=2 * banks[-1][name]["scale"])}]
    lengths = [40, 30, 7]
    x = torch.randn(sum(lengths) + 3, 2048, device=gpu)
    table = torch.arange(6, device=gpu, dtype=torch.int32).view(3, 2)
    out = []
    for b in (None, banks, twice):
        caches = paged.make_pools(NL, 6, device=gpu) if pages else kv8.make_caches(NL, 3, 64, device=gpu)
        out.append(prefill.prefill_packed(packed, *ln, x, lengths, caches, table=table if pages else None,
                                          adapters=None if b is None else (b, _ints(gpu, 1, -1, 0)))[:sum(lengths)].double())
    none, one, two = out
    assert torch.equal(none[40:70], one[40:70]) and bool((one - none)[:40].any()) and bool((one - none)[70:].any())
    largest = torch.maximum(torch.maximum(none.abs(), one.abs()), two.abs())
    assert bool(((two - none - 2 * (one - none)).abs() <= 2.0 ** -21 * largest).all())


def test_hidden_states_of_any_strides(gpu):
    """x as a transposed view gives the bits of its copy, with adapters too."""
    _, packed, _, ln = _weights(gpu, seed=5)
    x = torch.randn(2048, 45, device=gpu).t()
    adapters = _banks(gpu, 7), _ints(gpu, 0, 1)
    table = torch.arange(4, device=gpu, dtype=torch.int32).view(2, 2)
    a, b = (prefill.prefill_packed(packed, *ln, z, [30, 15], paged.make_pools(NL, 4, device=gpu), table=table, adapters=adapters)
            for z in (x, x.contiguous()))
    assert torch.equal(a, b)
