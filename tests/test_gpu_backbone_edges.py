"""Edges of ``prefill.prefill_packed`` and ``prefill.extend`` on the MI355X."""
import pytest
import torch

from flashact_amd import kv8, pi05, prefill
from tests.test_gpu_backbone import NL, _ints, _weights

pytestmark = pytest.mark.gpu


def test_tokens_behind_the_caches_end_are_not_real(gpu):
    """Those that fit get what they get alone: positions, keys and cache do not shift."""
    _, _, w4s, ln = _weights(gpu, seed=6)
    lens, filled = _ints(gpu, 30, 5, 32), kv8.make_caches(NL, 3, 32, device=gpu)
    prefill.extend(w4s, *ln, torch.randn(3, 20, 2048, device=gpu), filled, _ints(gpu, 0, 0, 0))
    x, runs = torch.randn(3, 4, 2048, device=gpu), []
    for count in (None, (9, 4, 1), (2, 4, 0)):
        caches = [{n: t.clone() for n, t in c.items()} for c in filled]
        runs.append((prefill.extend(w4s, *ln, x, caches, lens, None if count is None else _ints(gpu, *count)), caches))
    with pytest.raises(ValueError, match="count"):
        prefill.extend(w4s, *ln, x, caches, lens, _ints(gpu, 4))
    ref, want = runs[-1]
    for out, caches in runs[:-1]:
        assert torch.equal(out[0, :2], ref[0, :2]) and torch.equal(out[1], ref[1])
        assert all(torch.equal(a[n], b[n]) for a, b in zip(caches, want) for n in a)


def test_no_tokens(gpu):
    _, _, w4s, ln = _weights(gpu, seed=6)
    caches = kv8.make_caches(NL, 2, 32, device=gpu)
    assert prefill.extend(w4s, *ln, torch.zeros(2, 0, 2048, device=gpu), caches, _ints(gpu, 0, 3)).shape == (2, 0, 2048)


def test_caches_of_unequal_layers_are_refused(gpu):
    ln = [torch.zeros(NL, 2048, device=gpu) for _ in range(2)]
    packed = {k: torch.zeros(NL, n, m, dtype=torch.bfloat16, device=gpu)
              for k, n, m in (("wqkv", 2560, 2048), ("wo", 2048, 2048), ("wgu", 32768, 2048), ("wdn", 2048, 16384))}
    full = kv8.make_caches(NL, 2, 64, device=gpu)
    for other in (kv8.make_caches(1, 2, 32, device=gpu), kv8.make_caches(1, 3, 64, device=gpu)):
        caches = full[:1] + other
        with pytest.raises(ValueError, match="caches"):
            prefill.prefill_packed(packed, *ln, torch.zeros(50, 2048, device=gpu), [40, 10], caches)
        with pytest.raises(ValueError, match="caches"):
            prefill.extend([None] * NL, *ln, torch.zeros(2, 1, 2048, device=gpu), caches, _ints(gpu, 0, 0))


def test_two_samples_from_prompts_to_the_denoise_loops_caches(gpu):
    """Packed prompts, answers, and each sample's rows into its own caches of the denoise loop."""
    _, packed, w4s, ln = _weights(gpu, seed=7)
    lengths, cap = [20, 9], 40
    caches = kv8.make_caches(NL, batch=2, max_tokens=cap, device=gpu)
    prefill.prefill_packed(packed, *ln, torch.randn(sum(lengths), 2048, device=gpu), lengths, caches, prefix=[12, 9])
    lens = _ints(gpu, *lengths)
    for _ in range(3):
        prefill.extend(w4s, *ln, torch.randn(2, 1, 2048, device=gpu), caches, lens)
        lens += 1
    Lmax = pi05.lmax_for(cap, 50)
    kcache = torch.zeros(2, NL, Lmax, 256, dtype=torch.bfloat16, device=gpu)
    vtcache = torch.zeros(2, NL, 256, Lmax, dtype=torch.bfloat16, device=gpu)
    for l in range(NL):
        kv8.load(caches[l], lens, k=kcache[:, l, :, None], v=vtcache[:, l].transpose(1, 2)[:, :, None])
    for l in range(NL):
        k, v = kv8.load(caches[l], lens)
        for b, n in enumerate(lens.tolist()):
            assert torch.equal(kcache[b, l, :n], k[b, :n, 0]) and not kcache[b, l, n:].any()
            assert torch.equal(vtcache[b, l, :, :n].t(), v[b, :n, 0]) and not vtcache[b, l, :, n:].any()
