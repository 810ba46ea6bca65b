"""The adapters' definition in 64 bits, for the tests, with the bound of the kernels' error."""
import math

import torch

from flashact_amd import lora

F64 = torch.float64


def add(y, x, bank, index, gate=False):
    """(result, bound of the error before the result's rounding), fp64.

    h = A x is an fp32 sum of K exact products, taken in parts; it is multiplied by the scale (2^-24) and split into two values
    of the weights' type, which loses 2^-17 of it (fp16: less, or 2^-38 of the row's largest). B h is an fp32 sum of 2 rank products, and y is
    added to it. The gate multiplies an error by the slope of GeLU (below 1.13) and the input, and adds 2^-20 of its own.
    """
    out, bound = y.double().clone(), y.double().abs() * 2.0 ** -23
    x = x.double()
    for i, (a, b, s) in enumerate(lora.unpack(bank)):
        rows = (index == i).nonzero()[:, 0]
        if not rows.numel():
            continue
        a, b, xr = a.double(), b.double(), x[rows]
        h = xr @ a.t() * s
        eh = (a.shape[1] + 20) * 2.0 ** -24 * (xr.abs() @ a.abs().t()) * abs(s) + 2.0 ** -17 * h.abs() + 2.0 ** -36 * h.abs().amax(-1, keepdim=True)
        d = h @ b.t()
        out[rows] += d
        bound[rows] += (eh + (2 * a.shape[0] + 8) * 2.0 ** -24 * h.abs()) @ b.abs().t() + 2.0 ** -23 * d.abs()
    if gate:
        g, u, eg, eu = out[:, 0::2], out[:, 1::2], bound[:, 0::2], bound[:, 1::2]
        act = g / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))
        out = act * u
        bound = 1.13 * eg * u.abs() + act.abs() * eu + 1.13 * eg * eu + 2.0 ** -20 * out.abs() + 2.0 ** -20 * g.abs().clamp(max=1.0) * u.abs()
    return out, bound


def make(gen, device, adapters, rank, n, k, dtype, rows, ytype):
    """(y, x, bank): ranks differ where there are several adapters."""
    rand = lambda *s: torch.randn(*s, generator=gen, device=device)  # noqa: E731
    bank = lora.pack([(rand(max(1, rank - 3 * i), k) * k ** -0.5, rand(n, max(1, rank - 3 * i)) * 0.3, 0.5 + i) for i in range(adapters)],
                     dtype)
    return rand(rows, n).to(ytype), rand(rows, k).to(dtype), bank
