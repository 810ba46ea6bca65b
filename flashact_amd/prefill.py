"""pi0.5 prefix prefill on MI355X: the Gemma-2B-shaped backbone writes the K/V cache of the denoise loop.

``prefill`` replaces the reference's prefill and the cache hand-off after it: openpi's PaliGemma
forward with use_cache (benchmarks/pi05/eval_numerics.py:50-57), then compact_kv and the cache fill
(src/pi05/pack_weights.py:60-70; benchmarks/pi05/eval_numerics.py:83-87). It enqueues ONE
cooperative launch (C ABI ``fa_pi05_prefill``) that writes the RoPE'd keys into kcache rows
[0, Lp) and the transposed values into vtcache columns [0, Lp) of every layer, so the caches go
straight to ``pi05.launch`` with no copy in between.

``prefill_packed`` and ``extend`` run the same backbone where that launch does not reach: prompts of different lengths packed
one behind the other, with tokens that are causal behind a prefix that all see, and further tokens one by one (or a few)
behind what is cached. They keep keys and values in 8 bits (``kv8``), from where ``kv8.load`` fills the denoise loop's caches;
``extend`` reads the weights in 4 bits (``w4``).

Backbone shape: D = 2048, 8 query heads / 1 K/V head of 256, F = 16384 (GeLU-tanh gate), RMSNorm
eps 1e-6 scaled by (1 + w), RoPE base 10000 at positions 0..Lp-1, no mask inside the prefix.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, attention, kv8, pi05, w4

D, F, HD, H = 2048, 16384, 256, 8


def pack_backbone(wq, wk, wv, wo, wg, wu, wd) -> dict:
    """Natural [NL][out][in] backbone weights -> packed bf16 buffers (the expert's packing: q/k
    RoPE pairs adjacent, gate/up rows interleaved): {"wqkv", "wo", "wgu", "wdn"}."""
    p = pi05.pack_weights(wq, wk, wv, wo, wg, wu, wd)
    return {"wqkv": p["w1"], "wo": p["wo"], "wgu": p["w2"], "wdn": p["w3"]}


def pack_backbone_w4(packed: dict, group: int = 32) -> list:
    """``pack_backbone`` buffers -> per layer {"wqkv", "wo", "wgu", "wdn"} in 4 bits (``w4.quantize``), for ``extend``."""
    return [{k: w4.quantize(packed[k][l], group) for k in ("wqkv", "wo", "wgu", "wdn")}
            for l in range(int(packed["wqkv"].shape[0]))]


def rope_table(Lp: int, device=None):
    """cos/sin [Lp][128] for positions 0..Lp-1."""
    return pi05.rope_table(0, Lp, device=device)


_WS: dict = {}


def workspace(device, batch: int, Lp: int, Lmax: int) -> torch.Tensor:
    """Per-device cached workspace (zeroed once). One launch at a time may use it."""
    dev = torch.device(device)
    L = _lib.lib()
    nbytes = int(L.fa_pi05_prefill_workspace_bytes(batch, Lp, Lmax))
    if nbytes == 0:
        raise _lib.FlashActError(f"no prefill workspace for batch={batch} Lp={Lp} Lmax={Lmax}")
    key = dev.index if dev.index is not None else torch.cuda.current_device()
    ws = _WS.get(key)
    if ws is None or ws.numel() < nbytes:
        _WS.pop(key, None)
        raw = torch.empty(nbytes + 256, dtype=torch.uint8, device=dev)
        off = (-raw.data_ptr()) % 256
        ws = raw[off:off + nbytes]
        _lib.check(L.fa_pi05_workspace_init(ctypes.c_void_p(ws.data_ptr()), nbytes,
                                            ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)),
                   "fa_pi05_workspace_init")
        _WS[key] = ws
    return ws


def read_status(ws: torch.Tensor) -> int:
    return pi05.read_status(ws)


def release_buffers() -> None:
    """Drops the cached workspaces (they are re-created on the next launch)."""
    _WS.clear()


def _ptr(t, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def prefill(packed: dict, ln_in, ln_post, x, kcache, vtcache, rope_cos=None, rope_sin=None, *, stage_cycles=None,
            workspace_tensor=None, check_status=False):
    """Runs every backbone layer over the prefix and fills the caches in place.

    check_status=True waits for the launch and reads the kernel status; a non-zero status (a capped
    barrier wait expired, or the XCD placement differed, which leaves the caches unfinished)
    re-initialises the workspace and raises FlashActError.

    packed: ``pack_backbone`` output. ln_in, ln_post [NL][2048] fp32. x [B][Lp][2048] (or [Lp][2048])
    fp32: the hidden states entering layer 0. kcache [B][NL][Lmax][256] / vtcache [B][NL][256][Lmax]
    bf16 (or without the batch dimension). rope_cos/sin [Lp][128] (default: positions 0..Lp-1).
    """
    L = _lib.lib()
    for k in ("wqkv", "wo", "wgu", "wdn"):
        if packed[k].dtype != torch.bfloat16:
            raise TypeError(f"packed[{k!r}] must be bfloat16")
    if x.dtype != torch.float32 or ln_in.dtype != torch.float32 or ln_post.dtype != torch.float32:
        raise TypeError("x, ln_in and ln_post must be float32")
    if kcache.dtype != torch.bfloat16 or vtcache.dtype != torch.bfloat16:
        raise TypeError("kcache and vtcache must be bfloat16")
    batch = int(x.shape[0]) if x.dim() == 3 else 1
    Lp = int(x.shape[-2])
    NL = int(packed["wqkv"].shape[0])
    Lmax = int(kcache.shape[-2])
    if x.shape[-1] != D or kcache.shape[-1] != HD or vtcache.shape[-1] != Lmax:
        raise ValueError(f"shapes: x {tuple(x.shape)}, kcache {tuple(kcache.shape)}, vtcache {tuple(vtcache.shape)}")
    if kcache.numel() != batch * NL * Lmax * HD or vtcache.numel() != kcache.numel():
        raise ValueError("kcache / vtcache must hold [batch][NL][Lmax][256] / [batch][NL][256][Lmax]")
    dev = x.device
    if rope_cos is None or rope_sin is None:
        rope_cos, rope_sin = rope_table(Lp, device=dev)
    if rope_cos.shape != (Lp, HD // 2) or rope_sin.shape != (Lp, HD // 2):
        raise ValueError(f"rope tables must be [{Lp}][128]")
    wsp = workspace_tensor if workspace_tensor is not None else workspace(dev, batch, Lp, Lmax)
    a = _lib.PrefillArgs()
    a.weight_dtype = _lib.FA_DTYPE_BF16
    a.wqkv, a.wo, a.wgu, a.wdn = (_ptr(packed[k], k) for k in ("wqkv", "wo", "wgu", "wdn"))
    a.ln_in, a.ln_post = _ptr(ln_in, "ln_in"), _ptr(ln_post, "ln_post")
    a.rope_cos, a.rope_sin = _ptr(rope_cos, "rope_cos"), _ptr(rope_sin, "rope_sin")
    a.x = _ptr(x, "x")
    a.kcache, a.vtcache = _ptr(kcache, "kcache"), _ptr(vtcache, "vtcache")
    a.Lp, a.Lmax, a.num_layers, a.batch = Lp, Lmax, NL, batch
    if stage_cycles is not None and stage_cycles.numel() > 0:
        if stage_cycles.dtype != torch.int64 or stage_cycles.numel() < 16:
            raise TypeError("stage_cycles must be an int64 tensor with >= 16 entries")
        a.stage_cycles = _ptr(stage_cycles, "stage_cycles")
    a.workspace, a.workspace_bytes = wsp.data_ptr(), wsp.numel()
    stream = torch.cuda.current_stream(dev).cuda_stream
    _lib.check(L.fa_pi05_prefill(ctypes.byref(a), ctypes.c_void_p(stream)), "fa_pi05_prefill")
    if check_status:
        pi05.raise_on_status(wsp, torch.cuda.current_stream(dev), what="fa_pi05_prefill")


# ---------------------------------------------------------------- packed prompts, further tokens
def _norm(x, ln):
    return torch.nn.functional.rms_norm(x, (D,), 1.0 + ln, 1e-6).to(torch.bfloat16)


def _rope(pos, device):
    """cos, sin [..][128] of the positions' angles (the table of ``rope_table``, at any positions)."""
    inv = 1.0 / (10000.0 ** (torch.arange(0, HD, 2, dtype=torch.float32, device=device) / HD))
    a = pos.float()[..., None] * inv
    return a.cos()[..., None, :], a.sin()[..., None, :]


def _qkv(y, rope):
    """Rows [..][2560] of the packed projection (RoPE pairs adjacent) -> q [..][8][256], k and v [..][1][256], q and k turned
    and in split halves."""
    cos, sin = rope
    qk = y[..., :9 * HD].unflatten(-1, (9, HD // 2, 2)).float()
    a, b = qk[..., 0], qk[..., 1]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(y.dtype)
    return qk[..., :H, :], qk[..., H:, :], y[..., 9 * HD:].unflatten(-1, (1, HD))


def _check_backbone(ln_in, ln_post, layers, x, caches):
    if x.dtype is not torch.float32 or ln_in.dtype is not torch.float32 or ln_post.dtype is not torch.float32:
        raise TypeError("x, ln_in and ln_post must be float32")
    if x.shape[-1] != D or ln_in.shape != (layers, D) or ln_post.shape != (layers, D):
        raise ValueError(f"shapes: x {tuple(x.shape)}, ln_in {tuple(ln_in.shape)}, ln_post {tuple(ln_post.shape)}: need "
                         f"[..][{D}] and [{layers}][{D}]")
    if len(caches) != layers or any(c["v"].shape != caches[0]["v"].shape or c["v"].shape[1] != 1 or c["v"].shape[3] != HD for c in caches):
        raise ValueError(f"caches must be {layers} equal layers of kv8.make_caches with one K/V head of {HD}")


def prefill_packed(packed: dict, ln_in, ln_post, x, lengths, caches: list, prefix=None) -> torch.Tensor:
    """Runs the backbone over prompts of different lengths, packed one behind the other, into empty 8-bit caches.

    packed: ``pack_backbone`` output. x [T][2048] fp32: the hidden states entering layer 0 of prompt 0, then of prompt 1, and
    so on; lengths: their tokens (whole numbers, on the host; their sum is at most T, rows behind it are padding). prefix:
    how many of its first tokens all of a prompt sees, the others being causal (None: all, no mask in a prompt). caches:
    ``kv8.make_caches(layers, len(lengths), ...)``, filled from token 0 on. Returns the hidden states leaving the last
    layer [T][2048] fp32 (undefined in padding). The matrix products are the library's; the attention and the cache are
    ``attention.attend`` and ``kv8.store``.
    """
    layers = int(packed["wqkv"].shape[0])
    _check_backbone(ln_in, ln_post, layers, x, caches)
    lengths = [int(n) for n in lengths]
    prefix = lengths if prefix is None else [int(n) for n in prefix]
    if x.dim() != 2 or min(lengths, default=0) < 0 or sum(lengths) > x.shape[0] or len(prefix) != len(lengths):
        raise ValueError(f"x {tuple(x.shape)} must be [T][{D}] with T >= the sum of lengths {lengths}, and prefix {prefix} "
                         "as long as lengths")
    cap = caches[0]["v"].shape[2] * kv8.BLOCK
    if caches[0]["v"].shape[0] != len(lengths) or max(lengths, default=0) > cap:
        raise ValueError(f"caches of {caches[0]['v'].shape[0]} samples x {cap} tokens do not hold prompts of {lengths}")
    for k in ("wqkv", "wo", "wgu", "wdn"):
        if packed[k].dtype is not torch.bfloat16:
            raise TypeError(f"packed[{k!r}] must be bfloat16")
    dev, T = x.device, x.shape[0]
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    spans = attention.prefix_spans(t(lengths), t(prefix), T)
    rope = _rope(torch.arange(T, device=dev) - spans[:, 0], dev)
    zero, at = t([0]), [sum(lengths[:i]) for i in range(len(lengths))]
    for l in range(layers):
        q, k, v = _qkv(_norm(x, ln_in[l]) @ packed["wqkv"][l].t(), rope)
        for b, n in enumerate(lengths):
            if n:
                kv8.store({name: c[b:b + 1] for name, c in caches[l].items()}, k[None, at[b]:at[b] + n],
                          v[None, at[b]:at[b] + n], zero)
        o = attention.attend(q[None], k[None], v[None], spans)
        x = x + (o.view(T, H * HD) @ packed["wo"][l].t()).float()
        y = (_norm(x, ln_post[l]) @ packed["wgu"][l].t()).unflatten(-1, (F, 2)).float()
        h = (torch.nn.functional.gelu(y[..., 0], approximate="tanh") * y[..., 1]).to(torch.bfloat16)
        x = x + (h @ packed["wdn"][l].t()).float()
    return x


def extend(weights: list, ln_in, ln_post, x, caches: list, lens, count=None) -> torch.Tensor:
    """Runs the backbone over T further tokens of each sample behind its cached ones (answers token by token: T = 1).

    weights: ``pack_backbone_w4`` output. x [B][T][2048] fp32: the hidden states entering layer 0, B T <= 64. caches as
    ``prefill_packed`` leaves them; lens int32 [B] on the GPU: tokens cached so far, the positions of the new ones follow
    them; count int32 [B]: how many of the T are real (None: all, clamped to [0, T]); those behind the caches' end are not.
    The real tokens' keys and values are appended (the caller's lens grow by as many), each token sees all cached ones and the
    new ones up to itself. Returns the hidden states leaving the last layer [B][T][2048] fp32 (undefined where a token is not
    real). Nothing synchronises, and a captured graph serves every length.
    """
    _check_backbone(ln_in, ln_post, len(weights), x, caches)
    if x.dim() != 3 or x.shape[0] != caches[0]["v"].shape[0] or x.shape[0] * x.shape[1] > w4.MAX_ROWS:
        raise ValueError(f"x must be [B={caches[0]['v'].shape[0]}][T][{D}] with B T <= {w4.MAX_ROWS}, got {tuple(x.shape)}")
    B, T = int(x.shape[0]), int(x.shape[1])
    if count is not None and count.shape != lens.shape:
        raise ValueError(f"count must be [{B}] like lens, got {tuple(count.shape)} and {tuple(lens.shape)}")
    dev = x.device
    rope = _rope(lens[:, None] + torch.arange(T, device=dev), dev)
    room = (caches[0]["v"].shape[2] * kv8.BLOCK - lens).clamp(0, T)
    count = room if count is None else torch.minimum(count, room).clamp(min=0)
    after = lens + count
    x = x.reshape(B * T, D)
    for l, w in enumerate(weights):
        q, k, v = _qkv(w4.linear(_norm(x, ln_in[l]), w["wqkv"]).view(B, T, (H + 2) * HD), rope)
        kv8.store(caches[l], k, v, lens, count)
        o = kv8.attend(q, caches[l], after, count=count)
        x = w4.linear(o.view(B * T, H * HD), w["wo"], residual=x)
        h = w4.linear(_norm(x, ln_post[l]), w["wgu"], gate="gelu")
        x = w4.linear(h, w["wdn"], residual=x)
    return x.view(B, T, D)
