"""Rotary positions of one or several axes for the queries and keys of an attention layer (``nb200_rotary``).

One launch turns both tensors; its gradient is one launch as well.  Like the other operators of this package it always runs
the library's kernels: without a CUDA device or without the built library the call raises.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from .. import _cabi
from ..backend import resolve_backend

__all__ = ["rotary_embedding", "rotary_frequencies"]


def rotary_frequencies(sections: Sequence[int], *, base: float = 10000.0, device=None) -> torch.Tensor:
    """The usual frequencies, fp32 ``(sum(sections),)``: every axis has a ladder ``base ** (-j / pairs)`` over its own
    ``pairs``.  Formed in 64 bits."""
    if not sections or any(s < 0 for s in sections):
        raise ValueError(f"rotary_frequencies: sections must be the numbers of pairs of each axis; got {tuple(sections)}")
    if not base > 0:
        raise ValueError(f"rotary_frequencies: base must be positive; got {base}")
    rows = [torch.pow(torch.tensor(float(base), dtype=torch.float64), -torch.arange(s, dtype=torch.float64) / max(s, 1))
            for s in sections]
    return torch.cat(rows).float().to(device)


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor, *,
                     sections: Sequence[int] = (), interleaved: bool = False,
                     backend: str = "auto") -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(q, k)`` with their pairs turned by ``position * frequency``; new dense tensors.

    ``q`` is ``(..., heads, head_dim)``, ``k`` (or ``None``) the same with its own number of heads; fp32, bf16 or fp16.
    ``positions`` is ``(..., axes)`` (``(...)`` will do for one axis): int32, int64 or float32.  ``frequencies`` is fp32
    ``(pairs,)``; ``sections`` says how many of the pairs belong to each axis, in order (one axis by default).  A pair is
    elements ``(j, j + pairs)`` of a head, or ``(2 j, 2 j + 1)`` with ``interleaved``; elements from ``2 * pairs`` on pass
    unchanged.  Angles are as good at far positions as at near ones; the rotation is fp32, rounded once.  Differentiable in ``q`` and ``k``.
    """
    resolve_backend(backend)   # raises without a Blackwell device: there is no host path
    return _cabi.torch_ops().rotary(q, k, positions, frequencies, list(sections), bool(interleaved))
