"""ctypes binding of libflashact_mi355x.so (the C ABI declared in include/flashact_mi355x.h).

The library is built in-tree by ``flashact_amd.build`` (``__graft_entry__.build()``). There is
no fallback: if the shared library is missing or fails to load, every entry point raises.
"""
from __future__ import annotations

import ctypes
import functools
import os

import torch

from .build import LIB_PATH

ABI_VERSION = 2
STAGE_TICK_HZ = 100_000_000  # FA_STAGE_TICK_HZ: unit of the stage_cycles counters

FA_OK = 0
FA_DTYPE_BF16 = 0
FA_DTYPE_FP8_E4M3 = 1
FA_DTYPE_F16 = 2
FA_DTYPE_F32 = 3
FA_KSTATUS_SPIN_TIMEOUT = 1
FA_KSTATUS_XCD_MAP = 2
FA_KSTATUS_RANGE = 4


class FlashActError(RuntimeError):
    """A C-ABI entry point returned a non-zero status."""


class Pi05Args(ctypes.Structure):
    _fields_ = [
        ("weight_dtype", ctypes.c_int),
        ("w1", ctypes.c_void_p), ("wo", ctypes.c_void_p), ("w2", ctypes.c_void_p), ("w3", ctypes.c_void_p),
        ("s1", ctypes.c_void_p), ("so", ctypes.c_void_p), ("s2", ctypes.c_void_p), ("s3", ctypes.c_void_p),
        ("mods", ctypes.c_void_p), ("mod_final", ctypes.c_void_p),
        ("rope_cos", ctypes.c_void_p), ("rope_sin", ctypes.c_void_p),
        ("w_ain", ctypes.c_void_p), ("b_ain", ctypes.c_void_p), ("w_aout", ctypes.c_void_p), ("b_aout", ctypes.c_void_p),
        ("kvsrc_k", ctypes.c_void_p), ("kvsrc_v", ctypes.c_void_p), ("srows", ctypes.c_int),
        ("kcache", ctypes.c_void_p), ("vtcache", ctypes.c_void_p),
        ("Lp", ctypes.c_int), ("Lmax", ctypes.c_int), ("num_steps", ctypes.c_int), ("Tv", ctypes.c_int),
        ("num_layers", ctypes.c_int), ("batch", ctypes.c_int),
        ("x_t", ctypes.c_void_p), ("xt_rows", ctypes.c_int),
        ("stage_cycles", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
        ("trace", ctypes.c_void_p), ("trace_layer", ctypes.c_int),
        ("cache_dtype", ctypes.c_int), ("cache_shadow", ctypes.c_void_p), ("cache_shadow_bytes", ctypes.c_size_t),
    ]


class Ma2Args(ctypes.Structure):
    _fields_ = [
        ("weight_dtype", ctypes.c_int),
        ("w_qkv", ctypes.c_void_p), ("w_so", ctypes.c_void_p), ("w_cq", ctypes.c_void_p), ("w_co", ctypes.c_void_p),
        ("w_gu", ctypes.c_void_p), ("w_dn", ctypes.c_void_p),
        ("b_qkv", ctypes.c_void_p), ("b_so", ctypes.c_void_p), ("b_cq", ctypes.c_void_p), ("b_co", ctypes.c_void_p),
        ("b_gu", ctypes.c_void_p), ("b_dn", ctypes.c_void_p),
        ("mods", ctypes.c_void_p), ("mod_final", ctypes.c_void_p),
        ("rope_cos", ctypes.c_void_p), ("rope_sin", ctypes.c_void_p),
        ("w_ain", ctypes.c_void_p), ("b_ain", ctypes.c_void_p), ("w_aout", ctypes.c_void_p), ("b_aout", ctypes.c_void_p),
        ("kctx", ctypes.c_void_p), ("vtctx", ctypes.c_void_p),
        ("Lk", ctypes.c_int), ("Lkmax", ctypes.c_int), ("Tv", ctypes.c_int), ("adim", ctypes.c_int),
        ("num_steps", ctypes.c_int), ("num_layers", ctypes.c_int), ("batch", ctypes.c_int),
        ("x_t", ctypes.c_void_p), ("xt_rows", ctypes.c_int),
        ("stage_cycles", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
    ]


class PrefillArgs(ctypes.Structure):
    _fields_ = [
        ("weight_dtype", ctypes.c_int),
        ("wqkv", ctypes.c_void_p), ("wo", ctypes.c_void_p), ("wgu", ctypes.c_void_p), ("wdn", ctypes.c_void_p),
        ("ln_in", ctypes.c_void_p), ("ln_post", ctypes.c_void_p),
        ("rope_cos", ctypes.c_void_p), ("rope_sin", ctypes.c_void_p),
        ("x", ctypes.c_void_p), ("kcache", ctypes.c_void_p), ("vtcache", ctypes.c_void_p),
        ("Lp", ctypes.c_int), ("Lmax", ctypes.c_int), ("num_layers", ctypes.c_int), ("batch", ctypes.c_int),
        ("stage_cycles", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
    ]


class W4Args(ctypes.Structure):
    _fields_ = [
        ("dtype", ctypes.c_int), ("out_dtype", ctypes.c_int),
        ("x", ctypes.c_void_p), ("x_stride", ctypes.c_longlong), ("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p),
        ("rows", ctypes.c_int), ("n", ctypes.c_int), ("k", ctypes.c_int), ("group", ctypes.c_int),
        ("bias", ctypes.c_void_p), ("residual", ctypes.c_void_p), ("gate", ctypes.c_int), ("out", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
    ]


class Kv8RowsArgs(ctypes.Structure):
    _fields_ = [
        ("dtype", ctypes.c_int),
        ("k", ctypes.c_void_p), ("k_stride", ctypes.c_longlong * 4), ("v", ctypes.c_void_p), ("v_stride", ctypes.c_longlong * 4),
        ("cache_k", ctypes.c_void_p), ("cache_v", ctypes.c_void_p), ("cache_ks", ctypes.c_void_p), ("cache_vs", ctypes.c_void_p),
        ("start", ctypes.c_void_p), ("count", ctypes.c_void_p),
        ("batch", ctypes.c_int), ("tokens", ctypes.c_int), ("kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
        ("blocks", ctypes.c_int), ("zero_rest", ctypes.c_int),
    ]


class Kv8AttnArgs(ctypes.Structure):
    _fields_ = [
        ("dtype", ctypes.c_int), ("q", ctypes.c_void_p), ("q_stride", ctypes.c_longlong * 3),
        ("cache_k", ctypes.c_void_p), ("cache_v", ctypes.c_void_p), ("cache_ks", ctypes.c_void_p), ("cache_vs", ctypes.c_void_p),
        ("lens", ctypes.c_void_p), ("count", ctypes.c_void_p), ("slopes", ctypes.c_void_p),
        ("batch", ctypes.c_int), ("tokens", ctypes.c_int), ("heads", ctypes.c_int), ("kv_heads", ctypes.c_int),
        ("head_dim", ctypes.c_int), ("blocks", ctypes.c_int), ("causal", ctypes.c_int),
        ("scale", ctypes.c_float), ("softcap", ctypes.c_float), ("out", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
    ]


class SpanArgs(ctypes.Structure):
    _fields_ = [
        ("dtype", ctypes.c_int), ("q", ctypes.c_void_p), ("q_stride", ctypes.c_longlong * 3),
        ("k", ctypes.c_void_p), ("k_stride", ctypes.c_longlong * 3), ("v", ctypes.c_void_p), ("v_stride", ctypes.c_longlong * 3),
        ("spans", ctypes.c_void_p), ("slopes", ctypes.c_void_p),
        ("batch", ctypes.c_int), ("queries", ctypes.c_int), ("keys", ctypes.c_int), ("heads", ctypes.c_int),
        ("kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int), ("scale", ctypes.c_float), ("softcap", ctypes.c_float),
        ("out", ctypes.c_void_p), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
    ]


class PagedRowsArgs(ctypes.Structure):
    _fields_ = [
        ("dtype", ctypes.c_int), ("q", ctypes.c_void_p), ("q_stride", ctypes.c_longlong * 3), ("q_out", ctypes.c_void_p),
        ("k", ctypes.c_void_p), ("k_stride", ctypes.c_longlong * 4), ("v", ctypes.c_void_p), ("v_stride", ctypes.c_longlong * 4),
        ("pool_k", ctypes.c_void_p), ("pool_v", ctypes.c_void_p), ("table", ctypes.c_void_p), ("table_stride", ctypes.c_longlong),
        ("start", ctypes.c_void_p), ("count", ctypes.c_void_p), ("freqs", ctypes.c_void_p),
        ("batch", ctypes.c_int), ("tokens", ctypes.c_int), ("heads", ctypes.c_int), ("kv_heads", ctypes.c_int),
        ("head_dim", ctypes.c_int), ("pages", ctypes.c_int), ("table_pages", ctypes.c_int), ("rotary", ctypes.c_int),
        ("adjacent", ctypes.c_int), ("zero_rest", ctypes.c_int),
    ]


class PagedAttnArgs(ctypes.Structure):
    _fields_ = [
        ("dtype", ctypes.c_int), ("q", ctypes.c_void_p), ("q_stride", ctypes.c_longlong * 3),
        ("pool_k", ctypes.c_void_p), ("pool_v", ctypes.c_void_p), ("table", ctypes.c_void_p), ("table_stride", ctypes.c_longlong),
        ("lens", ctypes.c_void_p), ("count", ctypes.c_void_p), ("slopes", ctypes.c_void_p),
        ("batch", ctypes.c_int), ("tokens", ctypes.c_int), ("heads", ctypes.c_int), ("kv_heads", ctypes.c_int),
        ("head_dim", ctypes.c_int), ("pages", ctypes.c_int), ("table_pages", ctypes.c_int), ("causal", ctypes.c_int),
        ("scale", ctypes.c_float), ("softcap", ctypes.c_float), ("out", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
    ]


class LoraArgs(ctypes.Structure):
    _fields_ = [
        ("dtype", ctypes.c_int), ("y_dtype", ctypes.c_int), ("x", ctypes.c_void_p), ("x_stride", ctypes.c_longlong),
        ("a", ctypes.c_void_p), ("b", ctypes.c_void_p), ("scale", ctypes.c_void_p), ("index", ctypes.c_void_p),
        ("rows", ctypes.c_int), ("n", ctypes.c_int), ("k", ctypes.c_int), ("rank", ctypes.c_int), ("adapters", ctypes.c_int),
        ("gate", ctypes.c_int), ("y", ctypes.c_void_p), ("out", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
    ]


class TokenLogprobsArgs(ctypes.Structure):
    _fields_ = [
        ("dtype", ctypes.c_int), ("logits", ctypes.c_void_p), ("stride", ctypes.c_longlong), ("tokens", ctypes.c_void_p),
        ("wide_tokens", ctypes.c_int), ("scale", ctypes.c_float), ("rows", ctypes.c_int), ("vocabulary", ctypes.c_int),
        ("top", ctypes.c_int), ("logprob", ctypes.c_void_p), ("entropy", ctypes.c_void_p), ("top_tokens", ctypes.c_void_p),
        ("top_logprobs", ctypes.c_void_p), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
    ]


class DeviceInfo(ctypes.Structure):
    _fields_ = [("cus", ctypes.c_int), ("xcds", ctypes.c_int), ("lds_bytes", ctypes.c_int),
                ("coop_launch", ctypes.c_int), ("coop_max_blocks", ctypes.c_int), ("arch", ctypes.c_char * 64)]


# (name, restype, argtypes) of every symbol declared in include/flashact_mi355x.h
SYMBOLS = [
    ("fa_pi05_denoise", ctypes.c_int, [ctypes.POINTER(Pi05Args), ctypes.c_void_p]),
    ("fa_pi05_denoise_noalloc", ctypes.c_int,
     [ctypes.POINTER(Pi05Args), ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p)]),
    ("fa_pi05_workspace_bytes", ctypes.c_size_t, [ctypes.c_int, ctypes.c_int, ctypes.c_int]),
    ("fa_pi05_cache_shadow_bytes", ctypes.c_size_t, [ctypes.c_int, ctypes.c_int, ctypes.c_int]),
    ("fa_pi05_workspace_init", ctypes.c_int, [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]),
    ("fa_pi05_read_status", ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(ctypes.c_uint)]),
    ("fa_pi05_max_batch", ctypes.c_int, []),
    ("fa_ma2_flow", ctypes.c_int, [ctypes.POINTER(Ma2Args), ctypes.c_void_p]),
    ("fa_ma2_workspace_bytes", ctypes.c_size_t, [ctypes.c_int, ctypes.c_int, ctypes.c_int]),
    ("fa_ma2_workspace_init", ctypes.c_int, [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]),
    ("fa_ma2_read_status", ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(ctypes.c_uint)]),
    ("fa_ma2_max_batch", ctypes.c_int, []),
    ("fa_pi05_prefill", ctypes.c_int, [ctypes.POINTER(PrefillArgs), ctypes.c_void_p]),
    ("fa_pi05_prefill_workspace_bytes", ctypes.c_size_t, [ctypes.c_int, ctypes.c_int, ctypes.c_int]),
    ("fa_w4_linear", ctypes.c_int, [ctypes.POINTER(W4Args), ctypes.c_void_p]),
    ("fa_w4_workspace_bytes", ctypes.c_size_t, [ctypes.c_int, ctypes.c_int, ctypes.c_int]),
    ("fa_kv8_store", ctypes.c_int, [ctypes.POINTER(Kv8RowsArgs), ctypes.c_void_p]),
    ("fa_kv8_load", ctypes.c_int, [ctypes.POINTER(Kv8RowsArgs), ctypes.c_void_p]),
    ("fa_kv8_attention", ctypes.c_int, [ctypes.POINTER(Kv8AttnArgs), ctypes.c_void_p]),
    ("fa_kv8_attention_workspace_bytes", ctypes.c_size_t, [ctypes.c_int] * 6),
    ("fa_span_attention_workspace_bytes", ctypes.c_size_t, [ctypes.c_int] * 5),
    ("fa_span_attention", ctypes.c_int, [ctypes.POINTER(SpanArgs), ctypes.c_void_p]),
    ("fa_paged_append", ctypes.c_int, [ctypes.POINTER(PagedRowsArgs), ctypes.c_void_p]),
    ("fa_paged_load", ctypes.c_int, [ctypes.POINTER(PagedRowsArgs), ctypes.c_void_p]),
    ("fa_paged_attention", ctypes.c_int, [ctypes.POINTER(PagedAttnArgs), ctypes.c_void_p]),
    ("fa_paged_attention_workspace_bytes", ctypes.c_size_t, [ctypes.c_int] * 6),
    ("fa_lora_add", ctypes.c_int, [ctypes.POINTER(LoraArgs), ctypes.c_void_p]),
    ("fa_lora_workspace_bytes", ctypes.c_size_t, [ctypes.c_int] * 3),
    ("fa_token_logprobs", ctypes.c_int, [ctypes.POINTER(TokenLogprobsArgs), ctypes.c_void_p]),
    ("fa_token_logprobs_workspace_bytes", ctypes.c_size_t, [ctypes.c_int] * 4),
    ("fa_device_query", ctypes.c_int, [ctypes.c_int, ctypes.POINTER(DeviceInfo)]),
    ("fa_last_error", ctypes.c_char_p, []),
    ("fa_abi_version", ctypes.c_int, []),
]

# FA_DTYPE_* of a tensor's type
DTYPES = {torch.bfloat16: FA_DTYPE_BF16, torch.float16: FA_DTYPE_F16, torch.float32: FA_DTYPE_F32}

_lib = None


def lib() -> ctypes.CDLL:
    """Loads the in-tree shared library once; raises if it is absent (no fallback path)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FlashActError(f"{LIB_PATH} is missing: build it with `python -m flashact_amd.build` "
                                "(or __graft_entry__.build())")
        so = ctypes.CDLL(LIB_PATH)
        for name, res, args in SYMBOLS:
            fn = getattr(so, name)
            fn.restype = res
            fn.argtypes = args
        if so.fa_abi_version() != ABI_VERSION:
            raise FlashActError(f"ABI mismatch: library {so.fa_abi_version()} vs binding {ABI_VERSION}")
        _lib = so
    return _lib


def check(rc: int, what: str) -> None:
    if rc != FA_OK:
        msg = lib().fa_last_error()
        raise FlashActError(f"{what} failed (status {rc}): {msg.decode() if msg else ''}")


def run_on(index: int, fn, args, what: str) -> None:
    """Enqueues the C entry point `fn` on the current stream of GPU `index`, which need not be the current device."""
    if index == torch.cuda.current_device():
        rc = fn(ctypes.byref(args), torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(ctypes.byref(args), torch._C._cuda_getCurrentRawStream(index))
    if rc != FA_OK:
        check(rc, what)


def layout(t) -> tuple:
    """(type, shape, strides): what a call's checks depend on and their answers may be kept by."""
    return t.dtype, t.shape, t.stride()


def contiguous(lay) -> bool:
    """Whether a tensor of this ``layout`` is contiguous."""
    reach = 1
    for n, s in zip(reversed(lay[1]), reversed(lay[2])):
        if n > 1 and s != reach:
            return 0 in lay[1]
        reach *= n
    return True


def steps3(lay) -> tuple:
    """Strides of a ``layout``'s first three dimensions; those of size one, which are never stepped, as 0."""
    return tuple(s if n > 1 else 0 for n, s in zip(lay[1][:3], lay[2]))


def strides3(t) -> tuple:
    """Strides of a tensor's first three dimensions; those of size one, which are never stepped, as 0."""
    n, s = t.shape, t.stride()
    return (s[0] if n[0] > 1 else 0, s[1] if n[1] > 1 else 0, s[2] if n[2] > 1 else 0)


@functools.lru_cache(maxsize=1024)
def _layout(shape, stride) -> tuple:
    """(elements from the first to behind the last, whether two may be one) of a strided layout."""
    if 0 in shape:
        return 0, False
    reach, twice = 0, False
    for s, n in sorted((s, n) for s, n in zip(stride, shape) if n > 1):
        twice = twice or s <= reach
        reach += s * (n - 1)
    return reach + 1, twice


def ints(*sizes) -> tuple:
    """Sizes that the C structs hold as int, checked: ctypes would cut larger ones off."""
    if max(sizes) >= 1 << 31:
        raise ValueError(f"sizes {sizes} must be below 2^31")
    return sizes


def extent(lay) -> int:
    """Elements from the first to behind the last of a ``layout``."""
    return _layout(lay[1], lay[2])[0]


def overlap(a, b) -> bool:
    """Whether two tensors' memory ranges meet."""
    at, bt, na, nb = a.data_ptr(), b.data_ptr(), _layout(a.shape, a.stride())[0], _layout(b.shape, b.stride())[0]
    return na > 0 and nb > 0 and at < bt + nb * b.element_size() and bt < at + na * a.element_size()


def overlaps(a, others) -> bool:
    """Whether a's memory range meets one of the others' (None: none)."""
    at = a.data_ptr()
    end = at + _layout(a.shape, a.stride())[0] * a.element_size()
    if at == end:
        return False
    for b in others:
        if b is not None:
            bt = b.data_ptr()
            if bt < end and bt + _layout(b.shape, b.stride())[0] * b.element_size() > at:
                return True
    return False


def doubled(t) -> bool:
    """Whether two elements of a tensor may be one: a stride that does not step over all that smaller strides reach."""
    return _layout(t.shape, t.stride())[1]


def meet(a, b) -> bool:
    """Whether two tensors of one type have an element in common (or may have, where telling would take long)."""
    if not overlap(a, b):
        return False
    apart, odd = divmod(b.data_ptr() - a.data_ptr(), a.element_size())
    if odd:
        return True
    # sum of i * stride over a's dimensions less the same over b's = apart: by stride, the span of its factors
    spans = {}
    for t, low, high in ((a, 0, 1), (b, -1, 0)):
        for s, n in zip(t.stride(), t.shape):
            was = spans.get(s, (0, 0))
            spans[s] = (was[0] + low * (n - 1), was[1] + high * (n - 1))
    terms = sorted(((s, low, high) for s, (low, high) in spans.items() if s and (low or high)), reverse=True)
    least, most = [0], [0]  # what the terms behind one can add
    for s, low, high in reversed(terms):
        least.insert(0, least[0] + s * low)
        most.insert(0, most[0] + s * high)
    left = 10000

    def found(i, rest):
        nonlocal left
        if i == len(terms):
            return rest == 0
        s, low, high = terms[i]
        for c in range(max(low, -((most[i + 1] - rest) // s)), min(high, (rest - least[i + 1]) // s) + 1):
            left -= 1
            if left < 0 or found(i + 1, rest - c * s):
                return True
        return False

    return found(0, apart)
