"""The backbone over packed prompts and further tokens (``prefill.prefill_packed``, ``prefill.extend``) on the MI355X: the
8-bit cache, the spans' attention and the 4-bit products working together, as far as the action expert that reads the cache.

The prompts' cache is held against the fp32 oracle as the fused prefill's is (max-abs 4e-2, mean-abs 4e-3 at unit scale),
plus half a step of the codes (2^-4 of the value, 2^-10 of the scale's 448 below the normal range).

Hidden states are held against a 64-bit forward with the same weights (4-bit values that bf16 holds exactly) and the cache's
codes by their definition. Per layer five roundings to bf16 (normed rows twice, projection, attention, gated rows), 2^-8 of
their signal each: 0.02 a layer of what the layer adds. A bf16 rounding ahead of a code rounding moves at most 2^-8 / 2^-4 of the
values to the next code, an eighth off: sqrt(2^-4) 2^-3 = 0.03 of the attention. Two layers: 0.07, tested at 0.08 of the
2-norm of what the layers add.
"""
import numpy as np
import pytest
import torch

from flashact_amd import kv8, pi05, prefill, synthetic, w4
from tests import kv8_case
from tests import pi05_case as P
from tests import prefill_case as C

pytestmark = pytest.mark.gpu

NL, F64 = 2, torch.float64


def _ints(gpu, *v):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


@pytest.mark.parametrize("lengths", [(200, 129), (1, 300, 64), (77,)])
def test_packed_prompts_fill_the_cache_as_the_oracle(gpu, lengths):
    c = C.make_case(NL=NL, Lp=max(lengths), batch=1, seed=sum(lengths))
    g = C.gpu_weights(c, gpu)
    xs = [synthetic.prefix_inputs(7 + i, "cpu", batch=1, Lp=n)[0] for i, n in enumerate(lengths)]
    caches = kv8.make_caches(NL, len(lengths), max(lengths) + 5, device=gpu)
    x = torch.cat(xs + [torch.full((9, 2048), float("nan"))]).to(gpu)  # rows behind the last prompt are padding
    out = prefill.prefill_packed(g["packed"], g["ln_in"], g["ln_post"], x, lengths, caches)
    assert out.shape == x.shape and out[:sum(lengths)].isfinite().all()
    rows = [kv8.load(layer, _ints(gpu, *lengths), dtype=torch.float32) for layer in caches]
    for b, n in enumerate(lengths):
        one = dict(c, x=xs[b][None], Lp=n, batch=1)
        one["cos"], one["sin"] = pi05.rope_table(0, n)
        for want, which in zip(C.run_oracle(one), (0, 1)):
            got = np.stack([rows[l][which][b, :n, 0].cpu().numpy() for l in range(NL)])
            ref = want[0]
            code = 2.0 ** -4 * np.abs(ref) + 2.0 ** -10 * np.abs(ref).max() / 224
            err = np.abs(got - ref)
            print(f"packed {lengths} prompt {b} {'kv'[which]}: max {err.max():.4f} mean {err.mean():.5f}", flush=True)
            assert (err - code).max() <= 4e-2 and np.maximum(err - code, 0).mean() <= 4e-3


def test_packed_prompts_agree_with_the_fused_prefill(gpu):
    """One prompt without a mask: the same rows as the cooperative launch writes, but for the codes' rounding."""
    c = C.make_case(NL=NL, Lp=150)
    g = C.gpu_weights(c, gpu)
    kc, vt = C.run_gpu(c, gpu, g)
    caches = kv8.make_caches(NL, 1, 150, device=gpu)
    prefill.prefill_packed(g["packed"], g["ln_in"], g["ln_post"], c["x"][0].to(gpu), [150], caches)
    for l in range(NL):
        k, v = kv8.load(caches[l], _ints(gpu, 150), dtype=torch.float32)
        for got, ref in ((k[0, :150, 0], kc[0, l, :150].float()), (v[0, :150, 0], vt[0, l, :, :150].t().float())):
            err = (got - ref).abs() - 2.0 ** -4 * ref.abs() - 2.0 ** -10 * ref.abs().max() / 224
            assert float(err.max()) <= 4e-2 and float(err.clamp(min=0).mean()) <= 4e-3


# ---------------------------------------------------------------- further tokens
def _weights(gpu, seed=0):
    """Backbone weights that 4 bits hold exactly: random e2m1 values times 2^-8, the largest in every group of 32."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    table = torch.tensor(w4.E2M1 + tuple(-v for v in w4.E2M1), device=gpu)

    def w(n, k):
        x = table[torch.randint(0, 16, (NL, n, k), generator=g, device=gpu)]
        x[..., ::32] = 6.0
        return (x * torch.sign(torch.randn(NL, n, k, generator=g, device=gpu)) * 2.0 ** -8).bfloat16()

    nat = dict(wq=w(2048, 2048), wk=w(256, 2048), wv=w(256, 2048), wo=w(2048, 2048), wg=w(16384, 2048), wu=w(16384, 2048),
               wd=w(2048, 16384))
    ln = [torch.randn(NL, 2048, generator=g, device=gpu) * 0.1 for _ in range(2)]
    packed = prefill.pack_backbone(*nat.values())
    w4s = prefill.pack_backbone_w4(packed)
    for l in range(NL):
        for k in ("wqkv", "wo", "wgu", "wdn"):
            assert torch.equal(w4.dequantize(w4s[l][k]), packed[k][l].float())
    return nat, packed, w4s, ln


class _Reference:
    """The backbone in 64 bits, one sample at a time, with the cache's codes by their definition."""

    def __init__(self, nat, ln, length):
        self.w, self.ln = {k: v.double() for k, v in nat.items()}, [x.double() for x in ln]
        nb = (length + 31) // 32
        self.codes = [[torch.zeros(1, 1, nb * 32, 256, dtype=torch.uint8) for _ in range(2)] for _ in range(NL)]
        self.scales = [[torch.ones(1, 1, nb) for _ in range(2)] for _ in range(NL)]
        self.held = 0

    def _rope(self, y, pos):
        a = pos.double()[:, None] * (1.0 / 10000.0 ** (torch.arange(0, 256, 2, device=y.device).double() / 256))
        lo, hi = y[..., :128], y[..., 128:]
        cos, sin = a.cos()[:, None], a.sin()[:, None]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)

    def run(self, x, prefix=None):
        """prefix: a prompt's (attention over its own unrounded rows); None: further tokens (over the cache)."""
        x, n, dev = x.double(), x.shape[0], x.device
        pos = self.held + torch.arange(n, device=dev)
        norm = lambda v, g: v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6) * (1 + g)  # noqa: E731
        for l in range(NL):
            h = norm(x, self.ln[0][l])
            q = self._rope((h @ self.w["wq"][l].t()).view(n, 8, 256), pos)
            k = self._rope((h @ self.w["wk"][l].t()).view(n, 1, 256), pos)[:, 0]
            v = h @ self.w["wv"][l].t()
            for i, rows in enumerate((k, v)):
                kv8_case.store(self.codes[l][i], self.scales[l][i], rows.float()[None, :, None], [self.held], [n])
            if prefix is None:
                k, v = (kv8_case.values(self.codes[l][i], self.scales[l][i])[0, 0, :self.held + n].to(dev) for i in (0, 1))
            key = torch.arange(k.shape[0], device=dev)
            seen = (key <= pos[:, None]) | (key < (0 if prefix is None else prefix))
            s = torch.stack([q[:, i] @ k.t() for i in range(8)]) / 16
            o = torch.softmax(s.masked_fill(~seen, -float("inf")), -1) @ v
            x = x + o.transpose(0, 1).reshape(n, 2048) @ self.w["wo"][l].t()
            h = norm(x, self.ln[1][l])
            a = h @ self.w["wg"][l].t()
            a = 0.5 * a * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (a + 0.044715 * a ** 3)))
            x = x + (a * (h @ self.w["wu"][l].t())) @ self.w["wd"][l].t()
        self.held += n
        return x


def _close(out, ref, x):
    rel = float((out.double() - ref).norm() / (ref - x.double()).norm())
    print(f"2-norm off by {rel:.4f} of what the layers add", flush=True)
    assert rel <= 0.08


def test_answers_behind_packed_prompts(gpu):
    """Prompts of two lengths, one with causal tokens behind its prefix; then three tokens, one token, and a ragged step."""
    nat, packed, w4s, ln = _weights(gpu)
    lengths, prefix = [61, 37], [40, 37]
    caches = kv8.make_caches(NL, 2, 96, device=gpu)
    refs = [_Reference(nat, ln, 96) for _ in lengths]
    x = torch.randn(sum(lengths), 2048, device=gpu)
    out = prefill.prefill_packed(packed, *ln, x, lengths, caches, prefix)
    at = 0
    for n, p, r in zip(lengths, prefix, refs):
        _close(out[at:at + n], r.run(x[at:at + n], prefix=p), x[at:at + n])
        at += n
    lens = _ints(gpu, *lengths)
    for T, count in ((3, None), (1, None), (4, (4, 2)), (1, None)):
        x = torch.randn(2, T, 2048, device=gpu)
        n = [T, T] if count is None else count
        out = prefill.extend(w4s, *ln, x, caches, lens, None if count is None else _ints(gpu, *count))
        for b, r in enumerate(refs):
            _close(out[b, :n[b]], r.run(x[b, :n[b]]), x[b, :n[b]])
        lens = lens + _ints(gpu, *n)
    assert lens.tolist() == [r.held for r in refs]



def test_the_action_expert_reads_what_was_answered(gpu):
    """Prompt, answer, then the denoise loop on the cache's values: the same actions as from rows rounded by hand."""
    _, packed, w4s, ln = _weights(gpu, seed=2)
    cache = kv8.make_caches(NL, 1, 128, device=gpu)
    prefill.prefill_packed(packed, *ln, torch.randn(90, 2048, device=gpu), [90], cache, [80])
    lens = _ints(gpu, 90)
    for _ in range(3):
        prefill.extend(w4s, *ln, torch.randn(1, 1, 2048, device=gpu), cache, lens)
        lens += 1
    Lp, Lmax = 93, pi05.lmax_for(93, 50)
    kc = torch.zeros(NL, Lmax, 256, dtype=torch.bfloat16, device=gpu)
    vt = torch.zeros(NL, 256, Lmax, dtype=torch.bfloat16, device=gpu)
    for l in range(NL):
        kv8.load(cache[l], lens, k=kc[l][None, :, None], v=vt[l].t()[None, :, None])
        codes = kv8_case.rows_of(cache[l])
        for got, c, s in ((kc[l], codes[0], cache[l]["ks"]), (vt[l].t(), codes[1], cache[l]["vs"])):
            assert torch.equal(got[:Lp].cpu().double(), kv8_case.values(c, s)[0, 0, :Lp]) and not got[Lp:].any()
    case = P.make_case(NL=NL, Lp=Lp, Tv=50, S=2, seed=9)
    g = P.gpu_tensors(case, gpu)
    case["inp"]["kpre"] = kc[None, :, :Lp].cpu()
    case["inp"]["vpre"] = vt[None, :, :, :Lp].transpose(2, 3).cpu()
    g["caches"], g["Lmax"] = [(kc, vt)], Lmax
    st = P.parity(P.run_gpu(case, gpu, g)[0][:50], P.run_oracle(case)[0])
    print(f"actions behind an answer: {st}", flush=True)
    assert st["max_abs"] <= 2e-2 and st["mean_abs"] <= 2e-3


def test_refusals(gpu):
    ln = [torch.zeros(NL, 2048, device=gpu) for _ in range(2)]
    packed = {k: torch.zeros(NL, n, m, dtype=torch.bfloat16, device=gpu)
              for k, n, m in (("wqkv", 2560, 2048), ("wo", 2048, 2048), ("wgu", 32768, 2048), ("wdn", 2048, 16384))}
    caches, x = kv8.make_caches(NL, 2, 64, device=gpu), torch.zeros(20, 2048, device=gpu)
    for kw, err, text in ((dict(x=x.half()), TypeError, "float32"), (dict(x=x[:, :8]), ValueError, "shapes"),
                          (dict(lengths=[15, 6]), ValueError, "lengths"), (dict(lengths=[-1, 6]), ValueError, "lengths"),
                          (dict(prefix=[1]), ValueError, "prefix"), (dict(lengths=[1, 2, 3]), ValueError, "hold"),
                          (dict(x=torch.zeros(99, 2048, device=gpu), lengths=[65, 1]), ValueError, "hold"),
                          (dict(caches=caches[:1]), ValueError, "caches"),
                          (dict(caches=kv8.make_caches(NL, 2, 64, 2, 256, gpu)), ValueError, "caches"),
                          (dict(packed=dict(packed, wo=packed["wo"].half())), TypeError, "bfloat16")):
        with pytest.raises(err, match=text):
            prefill.prefill_packed(**{"packed": packed, "ln_in": ln[0], "ln_post": ln[1], "x": x, "lengths": [10, 10],
                                      "caches": caches, **kw})
    layers = [None] * NL
    for bad in (torch.zeros(2, 33, 2048, device=gpu), torch.zeros(3, 1, 2048, device=gpu), x):
        with pytest.raises(ValueError, match="x must be"):
            prefill.extend(layers, *ln, bad, caches, _ints(gpu, 0, 0))


def test_extend_clamps_counts(gpu):
    """A count past T is T, one below zero is none: the caches come out the same."""
    _, _, w4s, ln = _weights(gpu, seed=5)
    x, lens = torch.randn(2, 2, 2048, device=gpu), _ints(gpu, 0, 0)
    runs = []
    for count in ((2, 0), (9, -3)):
        caches = kv8.make_caches(NL, 2, 32, device=gpu)
        runs.append((prefill.extend(w4s, *ln, x, caches, lens, _ints(gpu, *count)), caches))
    assert torch.equal(runs[0][0][0], runs[1][0][0]) and runs[0][0][0].isfinite().all()
    assert all(torch.equal(a[n], b[n]) for a, b in zip(runs[0][1], runs[1][1]) for n in a)
