"""64-bit restatements of the root-mean-square norm and of a cache in 4 or 8 bits -- TEST INFRASTRUCTURE ONLY.

Written from the formulas, on torch tensors of any device.  Where rounding can change a number, the sums that bound by how much
come back beside it.
"""
from __future__ import annotations

import torch

GROUP = 32


# ---- norm --------------------------------------------------------------------------------------------------------------------
def stream_sum(x, residual):
    """The two streams' sum as it is stored: added in fp32, rounded to their type."""
    return x if residual is None else (x.float() + residual.float()).to(x.dtype)


def rms_norm(h, weight, eps):
    """``(y, n, s)``: the norm of rows ``h``, without its weight, and the factor of each row."""
    h = h.double()
    s = (h.square().mean(-1, keepdim=True) + eps) ** -0.5
    n = h * s
    return (n if weight is None else n * weight.double()), n, s


def rms_norm_grads(h, weight, eps, dy, dsum=None):
    """``(dx, its bound, dweight, its bound)``: relative errors ``u`` of all that is added change an entry by ``u`` times the bound."""
    _, n, s = rms_norm(h, weight, eps)
    dy = dy.double()
    g = dy if weight is None else dy * weight.double()
    mean = (g * n).mean(-1, keepdim=True)
    mean_bound = (g * n).abs().mean(-1, keepdim=True)
    dx, bound = s * (g - n * mean), s * (g.abs() + n.abs() * (mean.abs() + mean_bound))
    if dsum is not None:
        dx, bound = dx + dsum.double(), bound + dsum.double().abs()
    terms = (dy * n).reshape(-1, h.shape[-1])
    return dx, bound, terms.sum(0), terms.abs().sum(0)


def scales_of(y, group):
    """The fp32 scales of e4m3 codes, in 64 bits; ``group`` None: of rows."""
    parts = y.unflatten(-1, (-1, group or y.shape[-1]))
    return parts.abs().amax(-1).clamp(min=2.0 ** -100) / 448


# ---- cache -------------------------------------------------------------------------------------------------------------------
def quantize(x, bits):
    """``(codes, steps)`` of rows ``x``: codes as whole numbers (..., D), steps fp16 (..., D / 32).  The step is rounded to fp16, its
    inverse and the quotient to fp32, as the format says."""
    half = 1 << (bits - 1)
    parts = x.double().unflatten(-1, (-1, GROUP))
    high, low = parts.amax(-1), parts.amin(-1)
    step = (torch.where(high >= -low, high, low) / -half).clamp(-65504, 65504).half()
    finite = parts.isfinite().all(-1)
    step = torch.where(finite, step, torch.full_like(step, float("nan")))
    usable = finite & (step != 0)
    inverse = (1 / torch.where(usable, step, torch.ones_like(step)).double()).float().double()
    z = (parts * inverse[..., None]).float().double().nan_to_num(0.0)
    c = torch.where(usable[..., None], torch.round(z.clamp(-half, half - 1)), torch.zeros_like(z))
    return (c + half).long().flatten(-2), step


def packed_codes(codes, bits):
    """The bytes of a row: (8, groups, bits / 2), elements 4 j .. 4 j + 3 of a group together."""
    c = codes.unflatten(-1, (-1, 8, 4)).transpose(-3, -2)
    if bits == 4:
        c = c[..., 0::2] + 16 * c[..., 1::2]
    return c.flatten(-3).to(torch.uint8)


def values(packed, steps, bits):
    """What rows of bytes and their steps stand for, in 64 bits."""
    groups = steps.shape[-1]
    c = packed.long().unflatten(-1, (8, groups, bits // 2))
    if bits == 4:
        c = torch.stack([c % 16, c // 16], dim=-1).flatten(-2)
    return ((c - (1 << (bits - 1))).double() * steps.double()[..., None, :, None]).transpose(-3, -2).flatten(-3)


def cache_values(cache, bits):
    """The pages of a cache in few bits as 64-bit numbers: (k, v)."""
    return values(cache.k_codes, cache.k_steps, bits), values(cache.v_codes, cache.v_steps, bits)


def decode(q, k, v, table, lengths, scale):
    """``(out, sum p |v|, reach)`` over 64-bit pages; ``reach``: the largest sum of |scale q k| of any token, whose rounding errors
    are in the exponents."""
    H, Hk, page = q.shape[1], k.shape[1], k.shape[2]
    out, spread = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    reach = torch.zeros(q.shape[0], H, 1, dtype=torch.float64, device=q.device)
    for i, length in enumerate(lengths):
        if length == 0:
            continue
        at = torch.arange(length, device=q.device)
        pages, slots = table[i].long()[at // page], at % page
        for h in range(H):
            kk, vv = k[pages, h * Hk // H, slots], v[pages, h * Hk // H, slots]
            p = torch.softmax(scale * kk @ q[i, h].double(), 0)
            out[i, h], spread[i, h] = p @ vv, p @ vv.abs()
            reach[i, h] = (abs(scale) * kk.abs() @ q[i, h].double().abs()).max()
    return out, spread, reach
