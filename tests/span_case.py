"""Attention over spans of keys in plain torch and 64 bits, for the tests, with the bound of the kernel's error."""
import math

import torch

F64 = torch.float64


def attend(q, k, v, spans=None, scale=None, softcap=0.0, slopes=None):
    """(result, bound before the result's rounding), fp64; q [B][Tq][H][hd], k, v [B][Tk][Hkv][hd], spans [B][Tq][2].

    The bound: P is rounded to the values' type, eps / 2 relative (fp16 also 2^-25 absolute); a score's error d (hd + 8
    roundings of the running sum of |q k|, eight more of scaling and bias, 2^-21 cap of the tanh's exponential form) changes
    every weight by at most e^2d - 1 <= 3 d with its share of the sum; exp2 and the sums add 2^-20.
    """
    b, tq, hq, hd = q.shape
    tk, h, dev = k.shape[1], k.shape[2], q.device
    scale = hd ** -0.5 if scale is None else scale
    out, bound = torch.zeros(q.shape, dtype=F64, device=dev), torch.zeros(q.shape, dtype=F64, device=dev)
    key = torch.arange(tk, device=dev)
    pos = torch.arange(tq, device=dev) + tk - tq
    half = torch.finfo(q.dtype).eps / 2
    for i in range(b):
        sp = None if spans is None else (spans if spans.dim() == 2 else spans[i])
        seen = torch.ones(tq, tk, dtype=torch.bool, device=dev)
        if sp is not None:
            seen = (key >= sp[:, 0:1]) & (key < sp[:, 1:2])
        some = seen.any(-1, keepdim=True)
        for x in range(hq):
            qi, ki, vi = (t.double() for t in (q[i, :, x], k[i, :, x // (hq // h)], v[i, :, x // (hq // h)]))
            s = qi @ ki.t().contiguous() * scale
            d = (hd + 8) * 2.0 ** -24 * (qi.abs() @ ki.abs().t().contiguous()) * scale + 2.0 ** -21 * s.abs()
            if softcap:
                s = softcap * torch.tanh(s / softcap)
                d = d + 2.0 ** -21 * softcap
            if slopes is not None:
                bias = slopes[x].double() * (pos[:, None] - key).abs()
                s, d = s - bias, d + 2.0 ** -21 * bias.abs()
            p = torch.where(some, torch.softmax(s.masked_fill(~seen, -math.inf), -1), 0.0)
            vz = torch.where(torch.isfinite(vi), vi, 0.0)
            o = p @ vz
            for j in (~torch.isfinite(vi)).any(-1).nonzero().flatten().tolist():  # reaches who sees it
                o[seen[:, j]] += torch.where(torch.isfinite(vi[j]), 0.0, vi[j])
            out[i, :, x] = o
            d = d.masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            low = 2.0 ** -25 * (seen.double() @ vz.abs()) if q.dtype == torch.float16 else 0.0
            bound[i, :, x] = (p @ vz.abs()) * (half + 3 * d + 2.0 ** -20) + low
    return out, bound


def check(out, ref, bound):
    fine = torch.isfinite(ref)
    assert torch.equal(out.isnan(), ref.isnan())
    assert torch.equal(out[ref.isinf()].double(), ref[ref.isinf()])
    half = torch.finfo(out.dtype).eps / 2 * (ref.abs() + bound) + torch.finfo(out.dtype).tiny
    err = ((out.double() - ref).abs() - bound - half)[fine]
    assert bool((err <= 0).all()), float(err.max())
