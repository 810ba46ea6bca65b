"""The operators that serve many requests of the backbone at once, as measurable cases: one pass each through a public entry point.

Four operators make up the set:
  append    ``paged.append``: rows of keys and values into pages of 32 tokens that a table deals to the requests, keys
            (and queries) turned by their position on the way;
  attend    ``paged.attend``: attention of each request's newest tokens over its pages;
  adapters  ``lora.add``: the low-rank adapter of each row's own request beside a shared projection;
  logprobs  ``tokens.logprobs``: log probabilities of given tokens, with entropy and the best alternatives.
Layouts are the library's: pages k[pages][Hkv][hd/8][32][8] and v[pages][Hkv][4][hd][8] (token 8 i + j of a page is
[i][dim][j]) with a table[B][pages of a request] of page numbers; adapters a[adapters][K/8][rank][8] and
b[adapters][rank/8][N][8].
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
F32, F64 = torch.float32, torch.float64
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
PAGE = 32  # tokens of a page
BASE = 10000.0  # of the rotation


def _append(name, batch, tokens, start, heads=8, kv_heads=1, head_dim=256, rotary=1.0, adjacent=False, dtype="bf16"):
    return dict(name=name, kind="append", batch=batch, tokens=tokens, start=start, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, rotary=rotary, adjacent=adjacent, dtype=dtype)


def _attend(name, batch, tokens, shortest, longest, heads=8, kv_heads=1, head_dim=256, dtype="bf16", causal=True,
            softcap=0.0, bias=False):
    return dict(name=name, kind="attend", batch=batch, tokens=tokens, shortest=shortest, longest=longest, heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, causal=causal, softcap=softcap, bias=bias)


def _adapters(name, rows, n, k, rank, adapters, run=1, gate=False, dtype="bf16", y="bf16"):
    return dict(name=name, kind="adapters", rows=rows, n=n, k=k, rank=rank, adapters=adapters, run=run, gate=gate,
                dtype=dtype, y=y)


def _logprobs(name, rows, vocabulary, top, stride=0, scale=1.0, masked=0.0, dtype="bf16"):
    return dict(name=name, kind="logprobs", rows=rows, vocabulary=vocabulary, top=top, stride=max(stride, vocabulary),
                scale=scale, masked=masked, dtype=dtype)


def listed():
    return [
        # one step of sixteen requests: a token each behind its own prefix, pairs as the packed projection leaves them
        _append("append_token_b16", 16, 1, 989, adjacent=True),
        # the prompts of four requests, behind tokens that they have already; half of the dims turn
        _append("append_prompt_b4", 4, 2011, 13, heads=16, kv_heads=4, head_dim=128, rotary=0.5, dtype="f16"),
        # one token of one request over a prefix of three images and a prompt: latency counts
        _attend("attend_token_b1", 1, 1, 983, 983),
        # requests of very different age decoding together, grouped heads, capped scores and a distance bias
        _attend("attend_ragged_b48", 48, 1, 1, 8192, heads=16, kv_heads=4, head_dim=128, dtype="f16", softcap=30.0,
                bias=True),
        # the next piece of three long prompts: many new tokens over what is cached already
        _attend("attend_piece_b3", 3, 293, 1018, 4011, heads=8, kv_heads=2, head_dim=128),
        # a few requests with a very long history
        _attend("attend_long_b2", 2, 1, 130001, 131072),
        # one token of eight requests, each with an adapter of its own, beside the q/k/v projection: latency counts
        _adapters("adapters_token_b8", 8, 2560, 2048, 16, 8),
        # sixteen requests of five adapters, one without, beside the gated projection of the MLP
        _adapters("adapters_gate_b16", 16, 32768, 2048, 32, 5, gate=True, dtype="f16", y="f32"),
        # the prompts of several requests, packed, beside the MLP's way back into the residual stream
        _adapters("adapters_prompt", 1993, 2048, 16384, 16, 7, run=293, y="f32"),
        # one answer's next token out of a large vocabulary: latency counts
        _logprobs("logprobs_token_b1", 1, 262144, 8),
        # next tokens of forty-eight requests, a vocabulary of odd size, half of it ruled out, at a temperature
        _logprobs("logprobs_step_b48", 48, 99991, 20, stride=100000, scale=1.25, masked=0.5, dtype="f32"),
        # every token of a long text scored after the fact
        _logprobs("logprobs_text", 2011, 65537, 1),
    ]


def _size(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("append", "attend", "adapters", "logprobs"))
    dtype = rng.choice(("bf16", "f16"))
    if kind == "append":
        kv_heads, batch = rng.choice((1, 2, 4)), rng.choice((1, 2, 3, 4, 16))
        c = _append("", batch, _size(rng, 1, 2011 if batch <= 4 else 500), rng.choice((0, rng.randint(0, 4000))),
                    kv_heads * rng.choice((1, 2, 4)), kv_heads, rng.choice((64, 96, 128, 256)), rng.choice((1.0, 0.5)),
                    rng.random() < 0.5, dtype)
    elif kind == "attend":
        kv_heads = rng.choice((1, 2, 4, 8))
        head_dim = rng.choice((64, 96, 128, 256))
        longest = _size(rng, 1, 16384)
        group = rng.choice((1, 2, 3, 8))
        scores = (1 << 23) // (longest * kv_heads * group)  # what a piece of a prompt costs goes by its scores
        tokens = min(rng.choice((1, 1, 1, 2, 7, 50, _size(rng, 2, 300))), max(1, scores))
        batch = _size(rng, 1, max(1, min(48, (1 << 26) // (longest * kv_heads * head_dim), scores // tokens)))
        c = _attend("", batch, tokens, _size(rng, 1, longest), longest, kv_heads * group, kv_heads, head_dim, dtype,
                    rng.random() < 0.7, rng.choice((0.0, 30.0)), rng.random() < 0.3)
    elif kind == "adapters":
        rows, k = rng.choice((1, 2, 5, 16, 48, _size(rng, 1, 2011))), 8 * _size(rng, 8, 2048)
        n = 2 * _size(rng, 8, max(8, min(16384, (1 << 25) // max(rows, k))))
        c = _adapters("", rows, n, k, rng.choice((8, 16, 24, 32, 64)), rng.choice((1, 2, 5, 16)),
                      rng.choice((1, 1, 3, 200)), rng.random() < 0.3, dtype, rng.choice((dtype, "f32")))
    else:
        vocabulary = _size(rng, 2, 262144)
        c = _logprobs("", _size(rng, 1, max(1, min(2011, (1 << 27) // vocabulary))), vocabulary,
                      min(vocabulary, rng.choice((0, 1, 5, 20))), vocabulary + rng.choice((0, 0, 7, 64)),
                      rng.choice((1.0, 0.7, 1.25)), rng.choice((0.0, 0.0, 0.9)), rng.choice(("bf16", "f16", "f32")))
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs
def _lengths(count, shortest, longest):
    """`count` lengths from longest to shortest, spread over their logarithm."""
    return [int(round(longest * (shortest / longest) ** (i / max(1, count - 1)))) for i in range(count)]


def _slopes(heads):
    """2^(-8 (h + 1) / heads), the usual geometric series."""
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=F32, device=DEV)


def _pool(lens, kv_heads, head_dim, t, gen):
    """Pages of N(0, 1) in any order, a few more than the requests hold, and the table of who holds which."""
    need = [(n + PAGE - 1) // PAGE for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device=DEV).tolist()
    table, at = [], 0
    for n in need:  # behind a request's last page the table is empty
        table.append(order[at:at + n] + [-1] * (max(need) - n))
        at += n
    k = torch.randn(pages, kv_heads, head_dim // 8, PAGE, 8, generator=gen, device=DEV).to(t)
    v = torch.randn(pages, kv_heads, PAGE // 8, head_dim, 8, generator=gen, device=DEV).to(t)
    return {"k": k, "v": v}, torch.tensor(table, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, t = case["kind"], TYPES[case["dtype"]]
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    st = {"case": case}
    if kind == "append":
        b, tokens, hq, h, d = (case[x] for x in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
        # ragged: requests begin apart and end up to a fifth before the others
        count = [max(1, tokens - (i * tokens) // 5 // max(1, b - 1)) for i in range(b)]
        start = [max(0, case["start"] - 7 * i) for i in range(b)]
        st["start"], st["count"] = ints(start), ints(count)
        st["pool"], st["table"] = _pool([s + c for s, c in zip(start, count)], h, d, t, gen)
        qkv = rand(b, tokens, hq + 2 * h, d).to(t)  # one projection's output: views with the rows' stride
        st["q"], st["k"], st["v"] = qkv.split((hq, h, h), dim=2)
        rotary = int(d * case["rotary"]) // 2 * 2
        st["freqs"] = BASE ** (-torch.arange(0, rotary, 2, dtype=F64, device=DEV) / rotary)  # radians a position
    elif kind == "attend":
        b, tokens, hq, h, d = (case[x] for x in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
        lens = _lengths(b, case["shortest"], case["longest"])
        st["lens"] = ints(lens)
        st["pool"], st["table"] = _pool(lens, h, d, t, gen)
        st["q"] = rand(b, tokens, hq, d).to(t)
        st["slopes"] = _slopes(hq) if case["bias"] else None
    elif kind == "adapters":
        m, n, k, rank, many = (case[x] for x in ("rows", "n", "k", "rank", "adapters"))
        a, b = (rand(many, rank, k) * k ** -0.5).to(t), (rand(many, n, rank) * 0.1).to(t)
        st["bank"] = {"a": a.view(many, rank, k // 8, 8).transpose(1, 2).contiguous(),
                      "b": b.view(many, n, rank // 8, 8).transpose(1, 2).contiguous(),
                      "scale": 0.5 + torch.rand(many, generator=gen, device=DEV)}
        # requests of `run` rows each take the adapters in turn, and every so many have none
        row = torch.arange(m, device=DEV) // case["run"]
        st["index"] = torch.where(row % (many + 1) == many, -1, row % (many + 1)).to(torch.int32)
        st["x"], st["y"] = rand(m, k).to(t), rand(m, n).to(TYPES[case["y"]])
    else:
        m, n = case["rows"], case["vocabulary"]
        z = torch.empty(m, case["stride"], dtype=t, device=DEV)
        for i in range(0, m, 64):  # in pieces: the text's logits are large
            z[i:i + 64] = (rand(min(64, m - i), case["stride"]) * 3).to(t)
            if case["masked"]:
                out = torch.rand(min(64, m - i), case["stride"], generator=gen, device=DEV) < case["masked"]
                z[i:i + 64].masked_fill_(out, -math.inf)
        st["logits"] = z[:, :n]
        st["tokens"] = torch.randint(0, n, (m,), generator=gen, device=DEV)
    return st


# ---------------------------------------------------------------- the plain forms
def _turn(x, pos, freqs, adjacent):
    """Rows [B][T][heads][hd] -> fp32, the first 2 len(freqs) dims turned by their row's position [B][T], in split halves."""
    a = pos[..., None].double() * freqs
    a = torch.remainder(a, 2 * math.pi).float()[:, :, None]
    cos, sin = torch.cos(a), torch.sin(a)
    x, r = x.float(), 2 * freqs.shape[0]
    lo, hi = (x[..., 0:r:2], x[..., 1:r:2]) if adjacent else (x[..., :r // 2], x[..., r // 2:r])
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, x[..., r:]], -1)


def _append_plain(st):
    c, pool, t = st["case"], st["pool"], st["k"].dtype
    row = torch.arange(c["tokens"], device=DEV)
    pos = st["start"].long()[:, None] + row
    real = row < st["count"][:, None]
    q = _turn(st["q"], pos, st["freqs"], c["adjacent"])
    q = torch.where(real[..., None, None], q, 0.0).to(t)
    k, v = _turn(st["k"], pos, st["freqs"], c["adjacent"]).to(t)[real], st["v"][real]
    page = torch.gather(st["table"].long(), 1, (pos // PAGE).clamp(max=st["table"].shape[1] - 1))[real]
    slot = (pos % PAGE)[real]
    pool["k"][page, :, :, slot] = k.unflatten(-1, (-1, 8))
    pool["v"][page, :, slot // 8, :, slot % 8] = v
    return pool["k"], pool["v"], q


def _rows(pool, table):
    """The pages that a table names, as keys and values [B][Hkv][L][hd] in fp32."""
    at = table.long().clamp(min=0)
    k = pool["k"][at].float().permute(0, 2, 1, 4, 3, 5).flatten(4).flatten(2, 3)
    v = pool["v"][at].float().permute(0, 2, 1, 3, 5, 4).flatten(3, 4).flatten(2, 3)
    return k.contiguous(), v.contiguous()


def _attend_plain(st):
    c, q = st["case"], st["q"]
    k, v = _rows(st["pool"], st["table"])
    b, tokens, hq, d = q.shape
    h = c["kv_heads"]
    qg = q.float().view(b, tokens, h, hq // h, d).permute(0, 2, 3, 1, 4).reshape(b, h, -1, d)
    s = (qg @ k.transpose(-1, -2).contiguous()).view(b, hq, tokens, -1) * d ** -0.5
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    key = torch.arange(s.shape[-1], device=q.device)
    at = st["lens"].long()[:, None] - tokens + torch.arange(tokens, device=q.device)  # the queries' positions
    if c["bias"]:
        s = s - st["slopes"][:, None, None] * (at[:, None, :, None] - key).abs()
    last = at + 1 if c["causal"] else st["lens"].long()[:, None].expand(-1, tokens)
    s = torch.where((key < last[:, None, :, None]) & (at >= 0)[:, None, :, None], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), 0.0, m))
    p = (p / p.sum(-1, keepdim=True).clamp(min=1e-37)).view(b, h, -1, s.shape[-1])
    return (p @ v).view(b, hq, tokens, d).transpose(1, 2).contiguous().to(q.dtype)


def _adapters_plain(st):
    bank, x, index = st["bank"], st["x"].float(), st["index"]
    y = st["y"].float()
    for i in range(bank["scale"].shape[0]):
        a = bank["a"][i].float().transpose(0, 1).flatten(1)  # [rank][K]
        b = bank["b"][i].float().transpose(0, 1).flatten(1)  # [N][rank]
        d = (x @ a.t()) @ b.t() * bank["scale"][i]
        y = torch.where((index == i)[:, None], y + d, y)
    if st["case"]["gate"]:
        g, u = y[:, 0::2], y[:, 1::2]
        y = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g))) * u
        return y.to(st["x"].dtype)
    return y.to(st["y"].dtype)


def _logprobs_plain(st):
    c, tokens = st["case"], st["tokens"]
    z = st["logits"].float() * c["scale"]
    m = z.amax(-1, keepdim=True)
    d = z - torch.where(torch.isinf(m), 0.0, m)
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    total = torch.where(total == 0, 1.0, total)  # everything ruled out: log probabilities -inf, entropy 0
    logs = torch.log(total)
    entropy = logs[:, 0] - (torch.where(e > 0, d, 0.0) * e).sum(-1) / total[:, 0]
    logprob = torch.gather(d, 1, tokens[:, None])[:, 0] - logs[:, 0]
    if not c["top"]:
        return logprob, entropy
    # equal logits keep their order
    best, index = torch.sort(st["logits"].float(), dim=-1, descending=True, stable=True)
    index = index[:, :c["top"]]
    return logprob, entropy, index.to(torch.int32), torch.gather(d, 1, index) - logs


def run(state):
    c = state["case"]
    kind = c["kind"]
    if own:
        from flashact_amd import lora, paged, tokens
        if kind == "append":
            q = paged.append(state["pool"], state["table"], state["k"], state["v"], state["start"], state["count"],
                             q=state["q"], freqs=state["freqs"], adjacent=c["adjacent"])
            return state["pool"]["k"], state["pool"]["v"], q
        if kind == "attend":
            return paged.attend(state["q"], state["pool"], state["table"], state["lens"], softcap=c["softcap"],
                                slopes=state["slopes"], causal=c["causal"])
        if kind == "adapters":
            return lora.add(state["y"], state["x"], state["bank"], state["index"], gate="gelu" if c["gate"] else None)
        r = tokens.logprobs(state["logits"], state["tokens"], top=c["top"], scale=c["scale"])
        return (r.logprob, r.entropy, r.top_tokens, r.top_logprobs) if c["top"] else (r.logprob, r.entropy)
    return {"append": _append_plain, "attend": _attend_plain, "adapters": _adapters_plain,
            "logprobs": _logprobs_plain}[kind](state)


def work(case):
    kind = case["kind"]
    if kind == "append":
        d, hq, h = case["head_dim"], case["heads"], case["kv_heads"]
        b, tokens = case["batch"], case["tokens"]
        rows = sum(max(1, tokens - (i * tokens) // 5 // max(1, b - 1)) for i in range(b))
        return {"bytes": 4 * d * (rows * (hq + 2 * h)) + 2 * d * (b * tokens - rows) * hq,
                "flops": int(3 * rows * d * case["rotary"]) * (hq + h)}
    if kind == "attend":
        d, hq, h, tokens = case["head_dim"], case["heads"], case["kv_heads"], case["tokens"]
        lens = _lengths(case["batch"], case["shortest"], case["longest"])
        pairs = 0
        for n in lens:
            there = min(n, tokens)
            pairs += there * n - (there * (there - 1) // 2 if case["causal"] else 0)
        return {"bytes": sum(4 * n * h * d + 4 * -(-n // PAGE) for n in lens) + 4 * case["batch"] * tokens * hq * d,
                "flops": 4 * d * hq * pairs}
    if kind == "adapters":
        m, n, k, rank, many = (case[x] for x in ("rows", "n", "k", "rank", "adapters"))
        requests = -(-m // case["run"])
        used = min(many, requests)
        bare = sum(min(case["run"], m - i * case["run"]) for i in range(requests) if i % (many + 1) == many)
        y = 4 if case["y"] == "f32" else 2
        out = n if case["gate"] else y * n
        return {"bytes": 2 * (m - bare) * k + m * (y * n + out) + 2 * used * rank * (k + n),
                "flops": 2 * (m - bare) * rank * (k + n)}
    m, n = case["rows"], case["vocabulary"]
    return {"bytes": m * n * (4 if case["dtype"] == "f32" else 2) + m * (16 + 8 * case["top"]), "flops": 6 * m * n}


# ---------------------------------------------------------------- the definitions, in 64 bits
def _exact_append(st):
    c, pool = st["case"], st["pool"]
    d, r = c["head_dim"], 2 * st["freqs"].shape[0]
    keys = pool["k"].double().transpose(2, 3).flatten(3)  # [pages][Hkv][32][hd]
    values = pool["v"].double().transpose(3, 4).flatten(2, 3)
    j = torch.arange(r // 2, device=DEV)
    one, two = (2 * j, 2 * j + 1) if c["adjacent"] else (j, j + r // 2)
    f = torch.exp(-math.log(BASE) * 2 * j.double() / r)

    def turned(x, pos):  # [n][heads][hd]; as complex numbers
        z = torch.polar(torch.ones(pos.shape[0], r // 2, dtype=F64, device=DEV), pos.double()[:, None] * f)[:, None]
        z = z * torch.complex(x[..., one].double(), x[..., two].double())
        return torch.cat([z.real, z.imag, x[..., r:].double()], -1)

    q = torch.zeros(st["q"].shape, dtype=F64, device=DEV)
    for b in range(c["batch"]):
        n, s = int(st["count"][b]), int(st["start"][b])
        pos = s + torch.arange(n, device=DEV)
        q[b, :n] = turned(st["q"][b, :n], pos)
        page = st["table"][b].long()[pos // PAGE]
        keys[page, :, pos % PAGE] = turned(st["k"][b, :n], pos)
        values[page, :, pos % PAGE] = st["v"][b, :n].double()
    return (keys.unflatten(3, (d // 8, 8)).transpose(2, 3).contiguous(),
            values.unflatten(2, (PAGE // 8, 8)).transpose(3, 4).contiguous(), q)


def _exact_attend(st):
    c, q, pool = st["case"], st["q"], st["pool"]
    b, tokens, hq, d = q.shape
    group = hq // c["kv_heads"]
    out = torch.zeros(q.shape, dtype=F64, device=q.device)
    for i in range(b):
        n = int(st["lens"][i])
        there = min(n, tokens)
        at = torch.arange(n - there, n, device=q.device)
        token = torch.arange(n, device=q.device)
        page = st["table"][i].long()[token // PAGE]
        for x in range(c["kv_heads"]):
            k = pool["k"][page, x, :, token % PAGE].double().flatten(1)
            v = pool["v"][page, x, token % PAGE // 8, :, token % 8].double()
            for head in range(x * group, (x + 1) * group):
                s = q[i, tokens - there:, head].double() @ k.t() / math.sqrt(d)
                if c["softcap"]:
                    s = c["softcap"] * torch.tanh(s / c["softcap"])
                if c["bias"]:
                    s -= st["slopes"][head].double() * (at[:, None] - token).abs()
                if c["causal"]:
                    s.masked_fill_(token > at[:, None], -math.inf)
                out[i, tokens - there:, head] = torch.softmax(s, -1) @ v
    return out


def _exact_adapters(st):
    bank = st["bank"]
    y = st["y"].double()
    for i in range(bank["scale"].shape[0]):
        rows = (st["index"] == i).nonzero()[:, 0]
        if rows.numel():
            h = torch.einsum("mcj,crj->mr", st["x"][rows].double().unflatten(1, (-1, 8)), bank["a"][i].double())
            y[rows] += bank["scale"][i].double() * torch.einsum("mcj,cnj->mn", h.unflatten(1, (-1, 8)), bank["b"][i].double())
    if st["case"]["gate"]:
        g = y[:, 0::2]
        y = g / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * y[:, 1::2]
    return y


def _exact_logprobs(st):
    c = st["case"]
    out = []
    for i in range(0, c["rows"], 64):
        x = st["logits"][i:i + 64].double()
        z = x * c["scale"]
        z = torch.where((z == -math.inf).all(-1, keepdim=True), z, torch.log_softmax(z, -1))
        one = [z.gather(1, st["tokens"][i:i + 64, None])[:, 0], -(z.exp() * z.masked_fill(z.isinf(), 0.0)).sum(-1)]
        if c["top"]:
            # in place of a sort: take the largest one after the other, the first of equal ones
            index = torch.arange(x.shape[1], device=x.device)
            best = []
            for _ in range(c["top"]):
                top = x.nan_to_num(nan=-math.inf, neginf=-1e300)
                best.append(torch.where(top == top.amax(-1, keepdim=True), index, x.shape[1]).amin(-1))
                x.scatter_(1, best[-1][:, None], math.nan)
            best = torch.stack(best, -1)
            one += [best.to(torch.int32), z.gather(1, best)]
        out.append(one)
    return tuple(torch.cat(x) for x in zip(*out))


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "adapters": _exact_adapters,
            "logprobs": _exact_logprobs}[case["kind"]](st)
