"""Many requests served by the backbone at once on the MI355X: prompts into pages that requests share, further tokens with an
adapter for each request, log probabilities out of the last hidden states; against a 64-bit forward with the same weights.

Per layer seven roundings to bf16 (normed rows twice, projection, the adapter's sum on it, queries and keys, attention, gated rows), 2^-8 of
their signal each: 0.027 a layer of what the layer adds, 0.055 for two; tested at 0.06 of the 2-norm of what the layers add.
"""
import pytest
import torch

from flashact_amd import lora, paged, prefill, w4
from tests import tokens_case
from tests.test_gpu_backbone import F64, NL, _ints, _weights

pytestmark = pytest.mark.gpu


def _banks(gpu, seed, names=("wqkv", "wo", "wgu", "wdn"), adapters=2):
    gen = torch.Generator(device=gpu).manual_seed(seed)
    sizes = {"wqkv": (2560, 2048), "wo": (2048, 2048), "wgu": (32768, 2048), "wdn": (2048, 16384)}
    rand = lambda *s: torch.randn(*s, generator=gen, device=gpu)  # noqa: E731
    return [{m: lora.pack([(rand(4 + 8 * i, k) * k ** -0.5, rand(n, 4 + 8 * i) * 0.2, 1.0 + i) for i in range(adapters)])
             for m, (n, k) in sizes.items() if m in names} for _ in range(NL)]


class _Reference:
    """The backbone in 64 bits, one request at a time; packed weights, to which its adapter's product is added."""

    def __init__(self, packed, ln, banks, adapter, packed_after=None):
        self.packed, self.ln, self.banks, self.adapter = packed, [x.double() for x in ln], banks, adapter
        self.k, self.v = [[torch.zeros(0, 256, dtype=F64, device=ln[0].device) for _ in range(NL)] for _ in range(2)]

    def project(self, l, name, h):
        y = h @ self.packed[name][l].double().t()
        if self.adapter >= 0 and name in self.banks[l]:
            a, b, s = lora.unpack(self.banks[l][name])[self.adapter]
            y = y + s * (h @ a.double().t()) @ b.double().t()
        return y

    def turn(self, y, pos):  # pairs adjacent -> split halves
        a = pos.double()[:, None] * (10000.0 ** (-torch.arange(0, 256, 2, device=y.device).double() / 256))
        lo, hi = y[..., 0::2], y[..., 1::2]
        cos, sin = a.cos()[:, None], a.sin()[:, None]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)

    def run(self, x, prefix=0):
        x, n, dev = x.double(), x.shape[0], x.device
        pos = self.k[0].shape[0] + torch.arange(n, device=dev)
        norm = lambda v, g: v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6) * (1 + g)  # noqa: E731
        for l in range(NL):
            y = self.project(l, "wqkv", norm(x, self.ln[0][l])).view(n, 10, 256)
            qk = self.turn(y[:, :9], pos)
            self.k[l], self.v[l] = torch.cat([self.k[l], qk[:, 8]]), torch.cat([self.v[l], y[:, 9]])
            key = torch.arange(self.k[l].shape[0], device=dev)
            seen = (key <= pos[:, None]) | (key < prefix)
            s = torch.stack([qk[:, i] @ self.k[l].t() for i in range(8)]) / 16
            o = torch.softmax(s.masked_fill(~seen, -float("inf")), -1) @ self.v[l]
            x = x + self.project(l, "wo", o.transpose(0, 1).reshape(n, 2048))
            y = self.project(l, "wgu", norm(x, self.ln[1][l]))
            a = y[:, 0::2]
            a = 0.5 * a * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (a + 0.044715 * a ** 3)))
            x = x + self.project(l, "wdn", a * y[:, 1::2])
        return x


def _close(out, ref, x):
    rel = float((out.double() - ref).norm() / (ref - x.double()).norm())
    print(f"2-norm off by {rel:.4f} of what the layers add", flush=True)
    assert rel <= 0.06


@pytest.mark.parametrize("names", [("wqkv", "wo", "wgu", "wdn"), ("wqkv", "wdn"), ()])
def test_prompts_tokens_and_answers(gpu, names):
    """Three requests, one without an adapter: prompts, steps of one and more tokens, ragged ones, then what is answered."""
    _, packed, w4s, ln = _weights(gpu, seed=3)
    banks, which = _banks(gpu, 4, names), (1, -1, 0)
    adapters = (banks, _ints(gpu, *which)) if names else None
    lengths, prefix = [61, 37, 5], [40, 37, 0]
    refs = [_Reference(packed, ln, banks, a) for a in which]
    pools = paged.make_pools(NL, 12, device=gpu)
    order = torch.randperm(12, generator=torch.Generator().manual_seed(1)).tolist()
    table = torch.tensor([order[0:3] + [-1], order[3:6] + [-1], order[6:9] + [-1]], dtype=torch.int32, device=gpu)
    x = torch.randn(sum(lengths) + 4, 2048, device=gpu)  # the last rows are padding
    out = prefill.prefill_packed(packed, *ln, x, lengths, pools, prefix, table=table, adapters=adapters)
    at = 0
    for n, p, r in zip(lengths, prefix, refs):
        _close(out[at:at + n], r.run(x[at:at + n], prefix=p), x[at:at + n])
        at += n
    lens = _ints(gpu, *lengths)
    for T, count in ((3, None), (1, None), (4, (4, 2, 0)), (1, None)):
        x = torch.randn(3, T, 2048, device=gpu)
        n = [T] * 3 if count is None else count
        out = prefill.extend(w4s, *ln, x, pools, lens, None if count is None else _ints(gpu, *count), table=table, adapters=adapters)
        for b, r in enumerate(refs):
            if n[b]:
                _close(out[b, :n[b]], r.run(x[b, :n[b]]), x[b, :n[b]])
        lens = lens + _ints(gpu, *n)
    k, v = paged.load(pools[1], table, lens)
    for b, r in enumerate(refs):
        m = int(lens[b])
        for got, want in ((k, r.k[1]), (v, r.v[1])):
            assert float((got[b, :m, 0].double() - want).norm() / want.norm()) <= 0.06 and not got[b, m:].any()


def test_requests_share_a_prefix(gpu):
    """A common prompt's whole pages in two tables: both answer as if each had its own."""
    _, packed, w4s, ln = _weights(gpu, seed=6)
    x = torch.randn(64, 2048, device=gpu)
    pools = paged.make_pools(NL, 8, device=gpu)
    first = _ints(gpu, 5, 2, 0)[None]
    prefill.prefill_packed(packed, *ln, x, [64], pools, table=first)
    table = torch.cat([first, _ints(gpu, 5, 2, 7)[None]])
    new = torch.randn(2, 3, 2048, device=gpu)
    out = prefill.extend(w4s, *ln, new, pools, _ints(gpu, 64, 64), table=table)
    alone = paged.make_pools(NL, 8, device=gpu)
    for b in range(2):
        prefill.prefill_packed(packed, *ln, x, [64], alone, table=first)
        ref = _Reference(packed, ln, [{}] * NL, -1)
        ref.run(x, prefix=64)
        _close(out[b], ref.run(new[b]), new[b])


@pytest.mark.parametrize("four", [True, False])
def test_answer(gpu, four):
    """The final norm, the head and the log probabilities, against 64 bits: a logit is off by its operands' roundings (2^-9 each of
    |h| |w|), fp32 sums and, in bf16, its own (2^-9 of it); a log probability by at most twice the largest of a row."""
    gen = torch.Generator(device=gpu).manual_seed(1)
    v = 5003
    head = (torch.randn(v, 2048, generator=gen, device=gpu) * 0.05).bfloat16()
    ln, x = torch.randn(2048, generator=gen, device=gpu) * 0.1, torch.randn(2, 3, 2048, generator=gen, device=gpu)
    given = torch.randint(0, v, (2, 3), generator=gen, device=gpu)
    use = w4.quantize(head) if four else head
    w = (w4.dequantize(use) if four else head).double()
    h = x.double() * torch.rsqrt((x.double() ** 2).mean(-1, keepdim=True) + 1e-6) * (1 + ln.double())
    z = (h @ w.t()).view(6, v)
    off = (2.0 ** -8 * (h.abs() @ w.abs().t()).view(6, v) + (0 if four else 2.0 ** -9) * z.abs()).amax(-1)
    ref, _ = tokens_case.logprobs(z, given.view(6), 0, 0.7)
    got = prefill.answer(use, ln, x, given, top=3, scale=0.7)
    assert got.logprob.shape == (2, 3) and got.top_tokens.shape == (2, 3, 3)
    assert bool(((got.logprob.view(6).double() - ref["logprob"]).abs() <= 2 * 0.7 * off).all())
    best = prefill.answer(use, ln, x)
    assert torch.equal(best.logprob, best.top_logprobs[..., 0])
    lp = torch.log_softmax(z, -1)
    chosen = lp.gather(1, best.top_tokens.view(6, 1).long())[:, 0]
    assert bool((lp.amax(-1) - chosen <= 2 * off).all())
    assert torch.equal(best.top_tokens[..., 0], got.top_tokens[..., 0])


def test_without_table_and_adapters_nothing_changes(gpu):
    """The 8-bit path with adapters that are all none gives the bits of the call without."""
    from flashact_amd import kv8
    _, packed, w4s, ln = _weights(gpu, seed=8)
    x, new = torch.randn(50, 2048, device=gpu), torch.randn(2, 2, 2048, device=gpu)
    outs = []
    for adapters in (None, (_banks(gpu, 1, ("wqkv", "wo", "wdn")), _ints(gpu, -1, -1))):
        caches = kv8.make_caches(NL, 2, 96, device=gpu)
        a = prefill.prefill_packed(packed, *ln, x, [30, 20], caches, adapters=adapters)
        outs.append((a, prefill.extend(w4s, *ln, new, caches, _ints(gpu, 30, 20), adapters=adapters)))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
