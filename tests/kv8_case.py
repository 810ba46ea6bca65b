"""The 8-bit cache's definition in plain torch, for the tests: rows of codes, the store's rule, attention in 64 bits."""
import math

import torch

BLOCK = 32
F64 = torch.float64


def scale_for(amax: float) -> float:
    """The smallest power of two s with amax <= 448 s, within 2^-100 .. 2^120."""
    e = -100
    while e < 120 and amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def rows_of(cache):
    """uint8 codes of keys and values as rows [B][Hkv][L][hd] on the CPU."""
    k, v = cache["k"].cpu(), cache["v"].cpu()
    b, h, nb, hd, _ = v.shape
    return (k.transpose(3, 4).reshape(b, h, nb * BLOCK, hd).clone(), v.transpose(3, 4).reshape(b, h, nb * BLOCK, hd).clone())


def values(codes, scale):
    """Rows of codes and scales [B][Hkv][blocks] -> the values they stand for, fp64."""
    x = codes.contiguous().view(torch.float8_e4m3fn).float().double()
    return x * scale.cpu().double().repeat_interleave(BLOCK, 2)[..., None]


def store(codes, scale, new, start, count):
    """The store's rule on rows of codes [B][Hkv][L][hd] and scales, both changed in place; new [B][T][Hkv][hd]."""
    b, h, length, _ = codes.shape
    new = new.cpu().float()
    for i in range(b):
        s, n = int(start[i]), min(int(count[i]), new.shape[1], length - int(start[i]))
        if s < 0 or n <= 0:
            continue
        for x in range(h):
            for at in range(s // BLOCK * BLOCK, s + n, BLOCK):
                lo, hi = max(at, s), min(at + BLOCK, s + n)
                y = new[i, lo - s:hi - s, x]
                fine = y[torch.isfinite(y)].abs()
                to = scale_for(float(fine.max()) if fine.numel() else 0.0)
                old = float(scale[i, x, at // BLOCK])
                if lo > at:
                    to = max(to, old)
                    was = codes[i, x, at:lo].contiguous().view(torch.float8_e4m3fn).float()
                    codes[i, x, at:lo] = (was * (old / to)).to(torch.float8_e4m3fn).view(torch.uint8)
                z = torch.where(torch.isfinite(y), y / to, float("nan"))
                codes[i, x, lo:hi] = z.to(torch.float8_e4m3fn).view(torch.uint8)
                scale[i, x, at // BLOCK] = to


def attend(q, k, v, lens, count=None, scale=None, softcap=0.0, slopes=None, causal=True):
    """(result, bound of the error before the result's rounding), fp64, on q's device; k, v [B][Hkv][L][hd] fp64.

    The bound: P is rounded to fp16, 2^-12 relative or 2^-25 absolute; a score's error d (hd + 8 roundings of the running
    sum of |q k|, eight more of its scaling and of the bias, and of the cap's tanh, whose exponential form loses 2^-21 cap)
    changes every weight by at most e^2d - 1 <= 3 d with its share of the sum; exp2 and the sums add 2^-20.
    """
    b, t, hq, hd = q.shape
    h, dev = k.shape[1], q.device
    scale = hd ** -0.5 if scale is None else scale
    out, bound = torch.zeros(q.shape, dtype=F64, device=dev), torch.zeros(q.shape, dtype=F64, device=dev)
    for i in range(b):
        n = t if count is None else max(0, min(int(count[i]), t))
        length = max(0, min(int(lens[i]), k.shape[2]))
        first = max(0, n - length)  # the first query that is at a position
        if first >= n:
            continue
        pos = length - n + torch.arange(first, n, device=dev)
        key = torch.arange(length, device=dev)
        seen = key <= pos[:, None] if causal else torch.ones(n - first, length, dtype=torch.bool, device=dev)
        for x in range(hq):
            ki, vi, qi = k[i, x // (hq // h), :length], v[i, x // (hq // h), :length], q[i, first:n, x].double()
            s = qi @ ki.t() * scale
            d = (hd + 8) * 2.0 ** -24 * (qi.abs() @ ki.abs().t()) * abs(scale) + 2.0 ** -21 * s.abs()
            if softcap:
                s = softcap * torch.tanh(s / softcap)
                d = d + 2.0 ** -21 * softcap
            if slopes is not None:
                bias = slopes[x].double() * (pos[:, None] - key).abs()
                s, d = s - bias, d + 2.0 ** -21 * bias.abs()
            s = s.masked_fill(~seen, -math.inf)
            p = torch.softmax(s, -1)
            vz = torch.where(torch.isfinite(vi), vi, 0.0)
            o = p @ vz
            for j in (~torch.isfinite(vi)).any(-1).nonzero().flatten().tolist():  # a row with NaN reaches who sees it
                o[seen[:, j]] += torch.where(torch.isfinite(vi[j]), 0.0, math.nan)
            out[i, first:n, x] = o
            d = d.masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            bound[i, first:n, x] = (p @ vz.abs()) * (2.0 ** -12 + 3 * d + 2.0 ** -20) + 2.0 ** -25 * vz.abs().sum(0)
    return out, bound


def check(out, ref, bound):
    half = torch.finfo(out.dtype).eps / 2 * (ref.abs() + bound) + torch.finfo(out.dtype).tiny
    nan = ref.isnan()
    assert torch.equal(out.isnan(), nan)
    err = (out.double() - ref).abs() - bound - half
    assert bool((err.masked_fill(nan, 0.0) <= 0).all()), float(err.masked_fill(nan, 0.0).max())
