"""The paged cache's definition in plain torch, for the tests: where a token lies, the rotation, rows in and out."""
import math

import torch

PAGE = 32
F64 = torch.float64


def table_for(lens, pages, gen, width=None, device="cpu"):
    """A table of pages in any order for samples of `lens` tokens, -1 behind each one's last page."""
    need = [(n + PAGE - 1) // PAGE for n in lens]
    width = max(max(need), 1) if width is None else width
    order = torch.randperm(pages, generator=gen)[:sum(need)].tolist()
    rows = []
    for n in need:
        rows.append(order[:n] + [-1] * (width - n))
        order = order[n:]
    return torch.tensor(rows, dtype=torch.int32, device=device)


def filled(device, lens, kv_heads, hd, dtype, seed=0, width=None, spare=3):
    """A pool of N(0, 1) in every slot, and a table for samples of `lens` tokens."""
    gen = torch.Generator().manual_seed(seed)
    pages = sum((n + PAGE - 1) // PAGE for n in lens) + spare
    pool = {"k": torch.randn(pages, kv_heads, hd // 8, PAGE, 8, generator=gen).to(device, dtype),
            "v": torch.randn(pages, kv_heads, PAGE // 8, hd, 8, generator=gen).to(device, dtype)}
    return pool, table_for(lens, pages, gen, width, device)


def tokens_of(pool):
    """k and v as [pages][32][Hkv][hd]."""
    k = pool["k"].permute(0, 3, 1, 2, 4).flatten(3)
    v = pool["v"].permute(0, 2, 4, 1, 3).flatten(1, 2)
    return k, v


def rows_of(pool, table):
    """The tokens that a table names, [B][Hkv][L][hd] fp64 on the pool's device; of no page: zeros."""
    out = []
    for x in tokens_of(pool):
        y = torch.zeros(*table.shape, PAGE, *x.shape[2:], dtype=F64, device=x.device)
        there = (table >= 0) & (table < x.shape[0])
        y[there] = x[table[there].long()].double()
        out.append(y.flatten(1, 2).transpose(1, 2))
    return out


def turned(x, pos, freqs, adjacent):
    """Rows [n][heads][hd] at positions [n] -> (their first 2 len(freqs) dims turned, in 64 bits, and the bound of the error
    before the result's rounding).

    The bound: an angle's turns are rounded to 2^-26, 2^-23.3 radians; sine and cosine to four units, 2^-22; the two products
    and their sum to 2^-24 each: below 2^-21 of |x| + |y|. Either side's angle itself is rounded to 2^-53 up to three times.
    """
    x = x.double()
    if freqs is None:
        return x, torch.zeros_like(x)
    n, r = freqs.shape[0], 2 * freqs.shape[0]
    a = (pos.double()[:, None] * freqs)[:, None]
    lo, hi = (x[..., 0:r:2], x[..., 1:r:2]) if adjacent else (x[..., :n], x[..., n:r])
    y = torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin(), x[..., r:]], -1)
    b = (lo.abs() + hi.abs()) * (2.0 ** -21 + 6 * 2.0 ** -53 * a.abs())
    return y, torch.cat([b, b, torch.zeros_like(x[..., r:])], -1)


def append(pool, table, k, v, start, count, freqs, adjacent):
    """(keys, values, the keys' bound) [pages][32][Hkv][hd] fp64 of the pool after the append, on the CPU."""
    kt, vt = (x.cpu().double() for x in tokens_of(pool))
    bound = torch.zeros_like(kt)
    table, k, v = table.cpu(), k.cpu(), v.cpu()
    freqs = None if freqs is None else freqs.cpu()
    for b, s in enumerate(start):
        n = max(0, min(count[b], k.shape[1]))
        if s < 0 or n == 0:
            continue
        pos = s + torch.arange(n)
        kb, kbound = turned(k[b, :n], pos, freqs, adjacent)
        for i in range(n):
            at = (s + i) // PAGE
            page = int(table[b, at]) if at < table.shape[1] else -1
            if 0 <= page < kt.shape[0]:
                kt[page, (s + i) % PAGE], bound[page, (s + i) % PAGE] = kb[i], kbound[i]
                vt[page, (s + i) % PAGE] = v[b, i].double()
    return kt, vt, bound


def close(out, ref, bound):
    half = torch.finfo(out.dtype).eps / 2 * (ref.abs() + bound) + torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps
    err = (out.double() - ref).abs() - bound - half
    assert torch.equal(out.isnan(), ref.isnan())
    assert bool((err.nan_to_num(nan=-1.0) <= 0).all()), float(err.nan_to_num(nan=-1.0).max())


def attend_masked(q, k, v, seen, scale=None):
    """Softmax over what is seen, fp64, no caps or slopes: q [T][H][hd], k, v [Hkv][L][hd], seen [T][L]; zeros where nothing is.
    Values that are not finite are seen by nobody (a weight of zero times NaN would be NaN)."""
    v = torch.where(torch.isfinite(v), v, 0.0)
    group = q.shape[1] // k.shape[0]
    out = torch.zeros(q.shape, dtype=F64, device=q.device)
    for h in range(q.shape[1]):
        s = q[:, h].double() @ k[h // group].t() * (q.shape[2] ** -0.5 if scale is None else scale)
        p = torch.softmax(s.masked_fill(~seen, -math.inf), -1).nan_to_num(nan=0.0)
        out[:, h] = p @ v[h // group]
    return out
