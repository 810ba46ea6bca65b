"""Log probabilities in 64 bits, for the tests, with the bound of the kernel's error."""
import math

import torch


def logprobs(logits, tokens, top=0, scale=1.0):
    """({name: result}, {name: bound}), fp64; rows [M][V] without NaN or +inf.

    A term's exponent d = scale (x - m) is rounded three times (2^-22 |d|), exp2 to 2^-22: a weight p is off by (|d| + 1) 2^-21 of
    itself; a lane sums V / 256 terms (or fewer) and up to 100 sums meet: (V / 256 + 100) 2^-24. log s is off by as much, and
    2^-22 of itself; the entropy's t / s is a sum of p d with those errors and its own.
    """
    x = logits.double() * scale
    v = x.shape[1]
    m = x.amax(-1, keepdim=True)
    nothing = (m == -math.inf)[:, 0]
    d = (x - torch.where(torch.isinf(m), 0.0, m))
    e = d.exp()
    s = e.sum(-1)
    s = torch.where(nothing, 1.0, s)
    p, dz = e / s[:, None], torch.where(e > 0, d, 0.0)
    logs = s.log()
    terms = (v / 256 + 100) * 2.0 ** -24
    es = (p * (dz.abs() + 1)).sum(-1) * 2.0 ** -21 + terms
    elog = es + 2.0 ** -22 * (logs.abs() + 1)
    et = (p * dz.abs() * ((dz.abs() + 2) * 2.0 ** -21 + terms)).sum(-1) + (p * dz).sum(-1).abs() * es
    lp = d - logs[:, None]
    there = (tokens >= 0) & (tokens < v)
    got = lp.gather(1, tokens.clamp(0, v - 1).long()[:, None])[:, 0]
    out = {"logprob": torch.where(there, got, -math.inf), "entropy": torch.where(nothing, 0.0, logs - (p * dz).sum(-1))}
    # m is subtracted in fp32 and the difference scaled: 2^-22 of it
    one = lambda z: elog.view(-1, *[1] * (z.dim() - 1)) + 2.0 ** -22 * torch.where(torch.isinf(z), 0.0, z + logs.view(-1, *[1] * (z.dim() - 1))).abs()  # noqa: E731
    bound = {"logprob": one(out["logprob"]), "entropy": elog + et + 2.0 ** -22 * (out["entropy"].abs() + 1)}
    if top:
        best, index = torch.sort(logits.double(), dim=-1, descending=True, stable=True)
        out["top_tokens"] = index[:, :top].to(torch.int32)
        out["top_logprobs"] = lp.gather(1, index[:, :top])
        bound["top_logprobs"] = one(out["top_logprobs"])
    return out, bound


def check(got, ref, bound):
    for name, want in ref.items():
        x = getattr(got, name)
        if name == "top_tokens":
            assert x.dtype is torch.int32 and torch.equal(x, want), name
            continue
        assert x.dtype is torch.float32 and torch.equal(x.isinf(), want.isinf()) and not bool(x.isnan().any()), name
        fine = ~want.isinf()
        err = (x.double() - want)[fine].abs() - bound[name][fine] - 2.0 ** -24 * want[fine].abs()
        assert not err.numel() or float(err.max()) <= 0, (name, float(err.max()))
