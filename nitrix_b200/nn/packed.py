"""Attention over packed sequences of unequal length with grouped heads (``include/nitrix_b200_packed.h``)."""
from __future__ import annotations

from typing import Optional

import torch

from .. import _cabi
from ..backend import fallback, resolve_backend
from .attention import default_scale

__all__ = ["packed_attention"]

# why a pass leaves the tensor cores; True: the gradients alone
_REASONS = {
    False: "the fused tcgen05 kernels take head dim 64 or 128: bf16/fp16 with up to 64 query heads per key head and a "
           "positive scale, fp32 with up to 128 and 128 keys per sequence on average",
    True: "the fused tcgen05 kernels have the gradients of fp32 operands at head dim 64 with up to 64 query heads per key head, and "
          "those of more than 3 only where 16 blocks of 128 keys (32 from 8 query heads on), counted over the key heads, fill the GPU",
}


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, *,
                     offsets_k: Optional[torch.Tensor] = None, scale: Optional[float] = None, causal: bool = True,
                     backend: str = "auto") -> torch.Tensor:
    """Softmax attention within each of several sequences that lie one after the other.

    ``q`` is ``(tokens, heads, head_dim)``, ``k`` and ``v`` are ``(tokens, key heads, head_dim)``; query head ``h`` reads key
    head ``h // (heads // key heads)``.  Sequence ``i`` has the tokens ``offsets[i] .. offsets[i + 1]`` (int32, on the device);
    ``offsets_k`` where its keys are not as many as its queries.  With ``causal`` the last query of a sequence sees all its
    keys, each one before it one less.  A query that sees no key gives zeros and has no gradient; so do tokens before the
    first offset and behind the last.  Differentiable in ``q``, ``k`` and ``v``.

    bf16 and fp16 with head dim 64 or 128 run on the tensor cores, as do fp32 operands (three bf16 numbers each, good to 2^-20
    of a product; an infinity makes its rows NaN) of 128 keys per sequence or more on average: their forward pass, and their
    gradients at head dim 64.  A pass that the tensor cores do not take runs on the fp32 units, with one ``NitrixBackendFallback``
    warning per head layout and type when the forward pass is called.  That family sums everything in a fixed order and is what
    reproducibility mode uses.
    """
    resolved = resolve_backend(backend)
    kernel = _cabi.KERNEL_SIMT if resolved == "cuda-simt" else _cabi.KERNEL_AUTO
    factor = default_scale(q.shape[-1]) if scale is None else float(scale)
    out, gradients = _cabi.torch_ops().packed_attention(q, k, v, offsets, offsets_k, factor, bool(causal), kernel, False)
    if out is None:
        # (told per head layout: the number of tokens is another in every batch)
        fallback(function="packed_attention", requested=resolved, resolved="cuda-simt", reason=_REASONS[gradients],
                 shapes=(tuple(q.shape[1:]), tuple(k.shape[1:]), "gradients" if gradients else "forward"), dtype=q.dtype)
        out, _ = _cabi.torch_ops().packed_attention(q, k, v, offsets, offsets_k, factor, bool(causal), kernel, True)
    return out
