"""The operators that serve the backbone itself, as measurable cases: one pass each through a public entry point.

Four operators make up the set:
  linear   ``w4.linear``: products of a few rows of activations with 4-bit weights (e2m1 codes, a bf16 scale for
           each group of 32, 64 or 128 columns), with bias, residual or the gated form over pairs of rows;
  cache    ``kv8.store`` and ``kv8.load``: rows of keys and values into a cache of e4m3 codes with a power of two
           for each block of 32 tokens and head, and back;
  decode   ``kv8.attend``: attention of each sample's newest tokens over that cache;
  spans    ``attention.attend``: attention over packed prompts in which every query has its own span of keys.
Layouts are the library's: weights in tiles of 16 rows x 128 columns, codes[N/16][K/128][4][16][16] bytes (byte j of
[q][r] holds columns 32 (j / 4) + 8 q + 2 (j % 4) and the next, the lower nibble first) with scales[N/16][K/group][16];
cache blocks k[B][Hkv][L/32][hd/16][32][16] and v[B][Hkv][L/32][hd][32] with scales ks, vs[B][Hkv][L/32].
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
F32, F64 = torch.float32, torch.float64
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 32  # tokens of a cache block
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _linear(name, rows, n, k, group=32, dtype="bf16", epilogue="none"):
    return dict(name=name, kind="linear", rows=rows, n=n, k=k, group=group, dtype=dtype, epilogue=epilogue)


def _cache(name, batch, tokens, start, length, kv_heads=1, head_dim=256, dtype="bf16"):
    return dict(name=name, kind="cache", batch=batch, tokens=tokens, start=start, length=length, kv_heads=kv_heads,
                head_dim=head_dim, dtype=dtype)


def _decode(name, batch, tokens, shortest, longest, heads=8, kv_heads=1, head_dim=256, dtype="bf16", causal=True,
            softcap=0.0, bias=False):
    return dict(name=name, kind="decode", batch=batch, tokens=tokens, shortest=shortest, longest=longest, heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, causal=causal, softcap=softcap, bias=bias)


def _spans(name, documents, shortest, longest, prefix, heads=8, kv_heads=1, head_dim=256, dtype="bf16", softcap=0.0,
           bias=False, behind=0):
    return dict(name=name, kind="spans", documents=documents, shortest=shortest, longest=longest, prefix=prefix,
                heads=heads, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, softcap=softcap, bias=bias,
                behind=behind)


def listed():
    return [
        # one token of one request through the backbone's q/k/v projection: the smallest call, latency counts
        _linear("linear_token_qkv", 1, 2560, 2048),
        # five requests decoding together, the gated projection of the backbone's MLP
        _linear("linear_gate_b5", 5, 32768, 2048, group=64, dtype="f16", epilogue="gate"),
        # sixteen requests, the MLP's way back into the residual stream: few rows of weights, long sums
        _linear("linear_down_b16", 16, 2048, 16384, epilogue="residual"),
        # one step of sixteen requests: a token each behind its own cached prefix, blocks begun earlier
        _cache("cache_token_b16", 16, 1, 989, 1024),
        # the prompts of four requests into an empty cache
        _cache("cache_prompt_b4", 4, 2011, 0, 2048, kv_heads=4, head_dim=128, dtype="f16"),
        # one token of one request over a prefix of three images and a prompt: latency counts
        _decode("decode_token_b1", 1, 1, 983, 983),
        # requests of very different age decoding together, grouped heads, capped scores and a distance bias
        _decode("decode_ragged_b48", 48, 1, 1, 8192, heads=16, kv_heads=4, head_dim=128, dtype="f16", softcap=30.0,
                bias=True),
        # a chunk of action tokens that see the whole cache and each other
        _decode("decode_chunk_b4", 4, 50, 839, 1018, causal=False),
        # a few requests with a very long history
        _decode("decode_long_b2", 2, 1, 130001, 131072),
        # four prompts of different lengths, images first and seen by all, text causal behind them
        _spans("spans_prompts", 4, 293, 968, 0.8, behind=17),
        # image patches: every patch sees its own image, many heads of an odd size
        _spans("spans_images", 6, 256, 256, 1.0, heads=16, kv_heads=16, head_dim=72, dtype="f16"),
        # one long text, capped scores, heads that share keys
        _spans("spans_long", 1, 8191, 8191, 0.1, heads=16, kv_heads=4, head_dim=128, softcap=50.0),
    ]


def _size(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("linear", "cache", "decode", "spans"))
    dtype = rng.choice(("bf16", "f16"))
    if kind == "linear":
        epilogue = rng.choice(("none", "bias", "gate", "residual"))
        k = 8 * _size(rng, 8, 2048)
        n = 2 * _size(rng, 8, max(8, min(16384, (1 << 25) // k)))
        c = _linear("", rng.choice((1, 1, 2, 3, 5, 8, 13, 16)), n, k, rng.choice((32, 64, 128)), dtype, epilogue)
    elif kind == "cache":
        batch, kv_heads = rng.choice((1, 2, 3, 4)), rng.choice((1, 2, 4))
        tokens, start = _size(rng, 1, 2011), rng.choice((0, rng.randint(0, 31)))
        length = (start + tokens + 31) // 32 * 32
        c = _cache("", batch, tokens, start, length, kv_heads, rng.choice((64, 96, 128)), dtype)
    elif kind == "decode":
        kv_heads = rng.choice((1, 2, 4, 8))
        head_dim = rng.choice((64, 96, 128, 256))
        longest = _size(rng, 1, 16384)
        batch = _size(rng, 1, max(1, min(48, (1 << 27) // (2 * longest * kv_heads * head_dim))))
        c = _decode("", batch, rng.choice((1, 1, 1, 2, 7)), _size(rng, 1, longest), longest,
                    kv_heads * rng.choice((1, 2, 3, 8)), kv_heads, head_dim, dtype, rng.random() < 0.7,
                    rng.choice((0.0, 30.0)), rng.random() < 0.3)
    else:
        kv_heads, longest = rng.choice((1, 2, 4)), _size(rng, 1, 2048)
        c = _spans("", rng.choice((1, 2, 3)), _size(rng, 1, longest), longest, rng.choice((0.0, 0.3, 0.8, 1.0)),
                   kv_heads * rng.choice((1, 2, 4)), kv_heads, rng.choice((64, 72, 96, 128, 256)), dtype,
                   rng.choice((0.0, 50.0)), rng.random() < 0.3, rng.choice((0, 1, 40)))
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs
def _lengths(count, shortest, longest):
    """`count` lengths from longest to shortest, spread over their logarithm."""
    return [int(round(longest * (shortest / longest) ** (i / max(1, count - 1)))) for i in range(count)]


def _slopes(heads):
    """2^(-8 (h + 1) / heads), the usual geometric series."""
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=F32, device=DEV)


def _quantize4(w, group):
    """[N][K] weights -> packed codes and scales: scale = bf16(amax / 6) of each group, code the nearest e2m1."""
    n, k = w.shape
    np_, kp = (n + 15) // 16 * 16, (k + 127) // 128 * 128
    w = torch.nn.functional.pad(w.float(), (0, kp - k, 0, np_ - n))
    g = w.view(np_, kp // group, group)
    s = (g.abs().amax(-1) / 6.0).to(torch.bfloat16)
    y = (g / s.float().clamp(min=1e-30)[..., None]).view(np_, kp)
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)
    c = torch.bucketize(y.abs().contiguous(), edges).to(torch.uint8) | ((y < 0).to(torch.uint8) << 3)
    c = c.view(np_ // 16, 16, kp // 128, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 5, 6)  # tile, chunk, q, row, i, j, nibble
    codes = (c[..., 0] | (c[..., 1] << 4)).reshape(np_ // 16, kp // 128, 4, 16, 16).contiguous()
    return codes, s.view(np_ // 16, 16, kp // group).transpose(1, 2).contiguous()


def _quantize8(x):
    """[B][Hkv][L][hd] fp32 -> e4m3 codes [B][Hkv][L/32][32][hd] and scales [B][Hkv][L/32], a power of two each."""
    b, h, n, d = x.shape
    x = x.view(b, h, n // BLOCK, BLOCK, d)
    s = _scale_for(x.abs().amax((-1, -2)))
    return (x / s[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8), s


def _make_cache(batch, kv_heads, length, head_dim, gen):
    """A filled cache: keys and values N(0, 1), in the library's layout."""
    length = (length + BLOCK - 1) // BLOCK * BLOCK
    nb = length // BLOCK
    k = torch.randn(batch, kv_heads, length, head_dim, generator=gen, device=DEV)
    v = torch.randn(batch, kv_heads, length, head_dim, generator=gen, device=DEV)
    kc, ks = _quantize8(k)
    vc, vs = _quantize8(v)
    kc = kc.view(batch, kv_heads, nb, BLOCK, head_dim // 16, 16).transpose(3, 4).contiguous()
    return {"k": kc, "v": vc.transpose(-1, -2).contiguous(), "ks": ks, "vs": vs}


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, t = case["kind"], TYPES[case["dtype"]]
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    st = {"case": case}
    if kind == "linear":
        m, n, k, e = case["rows"], case["n"], case["k"], case["epilogue"]
        codes, scales = _quantize4(rand(n, k) * 0.02, case["group"])
        st["w"] = {"codes": codes, "scales": scales, "n": n, "k": k, "group": case["group"]}
        st["x"] = rand(m, k).to(t)
        st["bias"] = rand(n) if e == "bias" else None
        st["residual"] = rand(m, n) if e == "residual" else None
    elif kind == "cache":
        b, tokens, h, d = case["batch"], case["tokens"], case["kv_heads"], case["head_dim"]
        # ragged: samples begin and end up to a fifth before the others
        count = [max(1, tokens - (i * tokens) // 5 // max(1, b - 1)) for i in range(b)]
        start = [max(0, case["start"] - i) for i in range(b)]
        st["start"], st["count"] = ints(start), ints(count)
        st["lens"] = ints([s + c for s, c in zip(start, count)])
        st["cache"] = _make_cache(b, h, case["length"], d, gen)
        st["k"], st["v"] = rand(b, tokens, h, d).mul(3).to(t), rand(b, tokens, h, d).to(t)
    elif kind == "decode":
        b, tokens, hq, h, d = (case[x] for x in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
        lens = _lengths(b, case["shortest"], case["longest"])
        st["lens"] = ints(lens)
        st["cache"] = _make_cache(b, h, case["longest"], d, gen)
        st["q"] = rand(b, tokens, hq, d).to(t)
        st["slopes"] = _slopes(hq) if case["bias"] else None
    else:
        hq, h, d = case["heads"], case["kv_heads"], case["head_dim"]
        lens = _lengths(case["documents"], case["shortest"], case["longest"])
        total = sum(lens) + case["behind"]
        first, last = torch.zeros(total, dtype=torch.long), torch.zeros(total, dtype=torch.long)
        at = 0
        for n in lens:  # a document's first tokens are seen by all of it, those behind them by later ones
            first[at:at + n] = at
            last[at:at + n] = torch.maximum(torch.arange(at, at + n) + 1, torch.tensor(at + int(case["prefix"] * n)))
            at += n
        st["spans"] = torch.stack([first, last], -1).to(torch.int32).to(DEV)
        qkv = rand(total, hq + 2 * h, d).to(t)  # one projection's output: views with the rows' stride
        st["q"], st["k"], st["v"] = (x[None] for x in qkv.split((hq, h, h), dim=1))
        st["slopes"] = _slopes(hq) if case["bias"] else None
    return st


# ---------------------------------------------------------------- the plain forms
def _weights4(w):
    """Packed codes and scales -> [N][K] fp32."""
    nt, kc = w["codes"].shape[:2]
    c = torch.stack([w["codes"] & 15, w["codes"] >> 4], -1).view(nt, kc, 4, 16, 4, 4, 2).permute(0, 3, 1, 4, 2, 5, 6)
    c = c.reshape(nt * 16, kc * 128).long()
    x = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=c.device)[c]
    s = w["scales"].transpose(1, 2).reshape(nt * 16, -1).float().repeat_interleave(w["group"], 1)
    return (x * s)[:w["n"], :w["k"]]


def _linear_plain(st):
    e = st["case"]["epilogue"]
    y = st["x"].float() @ _weights4(st["w"]).t()
    if e == "bias":
        y = y + st["bias"]
    if e == "gate":
        a, b = y[:, 0::2], y[:, 1::2]
        y = 0.5 * a * (1 + torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a * a * a))) * b
    if e == "residual":
        return y + st["residual"]
    return y.to(st["x"].dtype)


def _scale_for(amax):
    """The smallest power of two s with amax <= 448 s, within 2^-100 .. 2^120."""
    m, x = torch.frexp(amax)
    e = torch.where(m > 0.875, x - 8, x - 9)
    e = torch.where(amax > 0, e, torch.full_like(e, -100)).clamp(-100, 120)
    return ((e + 127) << 23).view(F32)  # 2^e by its bits: pow and ldexp may round


def _rows(cache):
    """e4m3 codes of the cache's keys and values in rows, [B][Hkv][L][hd], and their values."""
    k, v = cache["k"], cache["v"]
    b, h, nb, d = v.shape[:4]
    k = k.transpose(3, 4).reshape(b, h, nb, BLOCK, d).view(torch.float8_e4m3fn).float()
    v = v.transpose(3, 4).contiguous().view(torch.float8_e4m3fn).float()
    return k, v


def _store_plain(codes, scale, new, start, count):
    """codes [B][Hkv][nb][32][hd] in fp32, scale [B][Hkv][nb], new [B][T][Hkv][hd] -> both after the store."""
    b, h, nb, _, d = codes.shape
    at = torch.arange(nb * BLOCK, device=codes.device)[None]
    row = at - start[:, None]
    fresh = (row >= 0) & (row < count[:, None])
    x = new.float()[torch.arange(b, device=codes.device)[:, None], row.clamp(0, new.shape[1] - 1)]
    x = torch.where(fresh[..., None, None], x, 0.0).permute(0, 2, 1, 3).reshape(b, h, nb, BLOCK, d)
    need = _scale_for(x.abs().amax((-1, -2)))
    fresh = fresh.view(b, 1, nb, BLOCK)
    earlier = (at < start[:, None]).view(b, 1, nb, BLOCK)
    to = torch.where(earlier.any(-1), torch.maximum(need, scale), need)
    to = torch.where(fresh.any(-1), to, scale)
    moved = torch.where(earlier[..., None], codes * (scale / to)[..., None, None], codes)
    moved = torch.where(fresh[..., None], x / to[..., None, None], moved)
    return moved.to(torch.float8_e4m3fn), to


def _cache_plain(st):
    cache, t = st["cache"], st["k"].dtype
    start, count = st["start"].long(), st["count"].long()
    k, v = _rows(cache)
    k, ks = _store_plain(k, cache["ks"], st["k"], start, count)
    v, vs = _store_plain(v, cache["vs"], st["v"], start, count)
    b, h, nb, _, d = k.shape
    cache["k"].copy_(k.view(torch.uint8).view(b, h, nb, BLOCK, d // 16, 16).transpose(3, 4))
    cache["v"].copy_(v.view(torch.uint8).transpose(3, 4))
    cache["ks"].copy_(ks)
    cache["vs"].copy_(vs)
    held = (torch.arange(nb * BLOCK, device=k.device)[None] < st["lens"][:, None])[:, :, None, None]
    kr = (k.float() * ks[..., None, None]).view(b, h, -1, d).transpose(1, 2)
    vr = (v.float() * vs[..., None, None]).view(b, h, -1, d).transpose(1, 2)
    return torch.where(held, kr, 0.0).to(t), torch.where(held, vr, 0.0).to(t)


def _softmax(s, seen):
    """Softmax over the last axis of what is seen; zeros where nothing is."""
    s = torch.where(seen, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), 0.0, m))
    return p / p.sum(-1, keepdim=True).clamp(min=1e-37)


def _decode_plain(st):
    c, q, cache = st["case"], st["q"], st["cache"]
    k, v = _rows(cache)
    k, v = k * cache["ks"][..., None, None], v * cache["vs"][..., None, None]
    b, tokens, hq, d = q.shape
    h = c["kv_heads"]
    k, v = k.view(b, h, -1, d), v.view(b, h, -1, d)
    qg = q.float().view(b, tokens, h, hq // h, d).permute(0, 2, 3, 1, 4).reshape(b, h, -1, d)
    s = (qg @ k.transpose(-1, -2).contiguous()).view(b, hq, tokens, -1) * d ** -0.5
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    key = torch.arange(s.shape[-1], device=q.device)
    at = st["lens"].long()[:, None] - tokens + torch.arange(tokens, device=q.device)  # the queries' positions
    if c["bias"]:
        s = s - st["slopes"][:, None, None] * (at[:, None, :, None] - key).abs()
    last = at + 1 if c["causal"] else st["lens"].long()[:, None].expand(-1, tokens)
    seen = (key < last[:, None, :, None]) & (at >= 0)[:, None, :, None]
    p = _softmax(s, seen).view(b, h, -1, s.shape[-1])
    o = (p @ v).view(b, hq, tokens, d).transpose(1, 2)
    return o.to(q.dtype)


def _spans_plain(st):
    c, hq, h = st["case"], st["case"]["heads"], st["case"]["kv_heads"]
    q, k, v = (st[x][0].float().transpose(0, 1) for x in "qkv")  # [heads][T][hd]
    n, d = q.shape[1:]
    s = (q.reshape(h, -1, d) @ k.transpose(-1, -2).contiguous()).view(hq, n, n) * d ** -0.5
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    at = torch.arange(n, device=q.device)
    if c["bias"]:
        s = s - st["slopes"][:, None, None] * (at[:, None] - at).abs()
    seen = (at >= st["spans"][:, 0:1]) & (at < st["spans"][:, 1:2])
    o = (_softmax(s, seen).view(h, -1, n) @ v.contiguous()).view(hq, n, d).transpose(0, 1)
    return o.to(st["q"].dtype)[None].contiguous()


def run(state):
    kind, c = state["case"]["kind"], state["case"]
    if own:
        from flashact_amd import attention, kv8, w4
        if kind == "linear":
            return w4.linear(state["x"], state["w"], bias=state["bias"], residual=state["residual"],
                             gate="gelu" if c["epilogue"] == "gate" else None)
        if kind == "cache":
            kv8.store(state["cache"], state["k"], state["v"], state["start"], state["count"])
            return kv8.load(state["cache"], state["lens"], dtype=state["k"].dtype)
        if kind == "decode":
            return kv8.attend(state["q"], state["cache"], state["lens"], softcap=c["softcap"], slopes=state["slopes"],
                              causal=c["causal"])
        return attention.attend(state["q"], state["k"], state["v"], state["spans"], softcap=c["softcap"],
                                slopes=state["slopes"])
    return {"linear": _linear_plain, "cache": _cache_plain, "decode": _decode_plain, "spans": _spans_plain}[kind](state)


def work(case):
    kind = case["kind"]
    if kind == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        out = {"gate": n, "residual": 8 * n}.get(case["epilogue"], 2 * n)  # bytes a row: half of n, or fp32 in and out
        return {"bytes": n * k // 2 + 2 * n * -(-k // case["group"]) + 2 * m * k + m * out
                + (4 * n if case["epilogue"] == "bias" else 0), "flops": 2 * m * n * k}
    if kind == "cache":
        row = case["kv_heads"] * case["head_dim"]
        new, held = case["batch"] * case["tokens"] * row, case["batch"] * (case["start"] + case["tokens"]) * row
        return {"bytes": 2 * (2 * new + new + held + 2 * held), "flops": 2 * 3 * new}
    d, hq, h = case["head_dim"], case["heads"], case["kv_heads"]
    if kind == "decode":
        lens = _lengths(case["batch"], case["shortest"], case["longest"])
        q = case["batch"] * case["tokens"] * hq * d
        return {"bytes": sum(2 * n * h * d + 8 * h * -(-n // BLOCK) for n in lens) + 4 * q,
                "flops": sum(4 * n * case["tokens"] * hq * d for n in lens)}
    lens = _lengths(case["documents"], case["shortest"], case["longest"])
    total = sum(lens) + case["behind"]
    pairs = sum(int(case["prefix"] * n) * n + (n - int(case["prefix"] * n)) * (n - int(case["prefix"] * n) + 1) // 2
                for n in lens)
    return {"bytes": 2 * total * d * (2 * hq + 2 * h) + 8 * total, "flops": 4 * d * hq * pairs}


# ---------------------------------------------------------------- the definitions, in 64 bits
def _exact_linear(st):
    w, c = st["w"], st["case"]
    codes, scales = w["codes"], w["scales"].double()
    n, k = w["n"], w["k"]
    i, j = torch.arange(n, device=codes.device)[:, None], torch.arange(k, device=codes.device)[None]
    byte = codes[i // 16, j // 128, j % 32 // 8, i % 16, j % 128 // 32 * 4 + j % 8 // 2].int()
    code = (byte >> (4 * (j % 2))) & 15
    e, f = (code >> 1) & 3, (code & 1).double()
    x = torch.where(e == 0, 0.5 * f, (1 + 0.5 * f) * _power(e - 1)) * (1 - 2 * (code >> 3).double())
    x = x * scales[i // 16, j // w["group"], i % 16]
    y = st["x"].double() @ x.t().contiguous()
    if c["epilogue"] == "bias":
        y += st["bias"].double()
    if c["epilogue"] == "residual":
        y += st["residual"].double()
    if c["epilogue"] == "gate":
        g = y[:, 0::2]
        y = g / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * y[:, 1::2]
    return y


def _power(e):
    """2^e for whole e, exactly."""
    return ((e.long() + 1023) << 52).view(F64)


def _nearest_e4m3(y):
    """The e4m3 value nearest to y (ties to the even one), |y| <= 448."""
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = _power(e - 3)
    return torch.round(y / step) * step


def _e4m3_value(codes):
    c = codes.int()
    e, f = (c >> 3) & 15, (c & 7).double()
    return torch.where(e == 0, f * 2.0 ** -9, (1 + f / 8) * _power(e - 7)) * (1 - 2 * (c >> 7).double())


def _exact_cache(st):
    cache, out = st["cache"], []
    length = cache["v"].shape[2] * BLOCK
    for codes, scale, new in ((cache["k"].transpose(3, 4).flatten(4), cache["ks"], st["k"]),
                              (cache["v"].transpose(3, 4), cache["vs"], st["v"])):
        held = _e4m3_value(codes).flatten(2, 3)  # [B][Hkv][L][hd]
        rows = torch.zeros(held.shape[0], length, *held.shape[1::2], dtype=F64, device=held.device)
        for b in range(held.shape[0]):
            s, n = int(st["start"][b]), int(st["count"][b])
            for at in range(0, s + n, BLOCK):
                end = min(at + BLOCK, s + n)
                old = held[b, :, at:end] * scale[b, :, at // BLOCK, None, None].double()
                if end > s:
                    lo = max(at, s)
                    x = new[b, lo - s:end - s].transpose(0, 1).double()
                    x_max = x.abs().amax((-1, -2)).clamp(min=448 * 2.0 ** -100)
                    to = _power(torch.ceil(torch.log2(x_max / 448) - 1e-9))  # inputs of 24 bits: no border is nearer
                    if lo > at:
                        to = torch.maximum(to, scale[b, :, at // BLOCK].double())
                    old = torch.cat([old[:, :lo - at], x], 1) / to[:, None, None]
                    old = _nearest_e4m3(old) * to[:, None, None]
                rows[b, at:end] = old.transpose(0, 1)
        out.append(rows)
    return tuple(out)


def _exact_attention(q, k, v, first, last, at, softcap, slopes):
    """One head: q [T][hd], k, v [N][hd] in 64 bits; query i at position at[i] sees the keys first[i] .. last[i] - 1."""
    j = torch.arange(k.shape[0], device=q.device)
    s = q @ k.t() / math.sqrt(q.shape[-1])
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if slopes is not None:
        s -= slopes.double() * (at[:, None] - j).abs()
    s.masked_fill_((j < first[:, None]) | (j >= last[:, None]), -math.inf)
    return torch.nan_to_num(torch.softmax(s, -1), nan=0.0) @ v


def _exact_decode(st):
    c, q, cache = st["case"], st["q"], st["cache"]
    b, tokens, hq, d = q.shape
    out = torch.zeros(q.shape, dtype=F64, device=q.device)
    for i in range(b):
        n = int(st["lens"][i])
        at = n - tokens + torch.arange(tokens, device=q.device)
        last = torch.where(at < 0, 0, at + 1 if c["causal"] else n)
        for kv in range(c["kv_heads"]):
            k = _e4m3_value(cache["k"][i, kv].transpose(1, 2).flatten(2)) * cache["ks"][i, kv, :, None, None].double()
            v = _e4m3_value(cache["v"][i, kv].transpose(1, 2)) * cache["vs"][i, kv, :, None, None].double()
            k, v = k.flatten(0, 1)[:n], v.flatten(0, 1)[:n]
            for head in range(kv * (hq // c["kv_heads"]), (kv + 1) * (hq // c["kv_heads"])):
                out[i, :, head] = _exact_attention(q[i, :, head].double(), k, v, torch.zeros_like(at), last, at,
                                                   c["softcap"], st["slopes"][head] if c["bias"] else None)
    return out


def _exact_spans(st):
    c, q = st["case"], st["q"]
    at = torch.arange(q.shape[1], device=q.device)
    out = torch.zeros(q.shape, dtype=F64, device=q.device)
    for head in range(c["heads"]):
        kv = head // (c["heads"] // c["kv_heads"])
        out[0, :, head] = _exact_attention(q[0, :, head].double(), st["k"][0, :, kv].double(),
                                           st["v"][0, :, kv].double(), st["spans"][:, 0], st["spans"][:, 1], at,
                                           c["softcap"], st["slopes"][head] if c["bias"] else None)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"linear": _exact_linear, "cache": _exact_cache, "decode": _exact_decode,
            "spans": _exact_spans}[case["kind"]](st)
