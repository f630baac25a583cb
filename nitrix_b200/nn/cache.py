"""A paged key / value cache, and the attention of one new token per sequence over it (``include/nitrix_b200_cache.h``).

The cache of a layer is a pool of pages and a table that says which pages hold which sequence's tokens.  All bookkeeping runs
on the device: no call waits for the GPU, and a generation step can be captured into a CUDA graph.

A :class:`PagedCache` is a value: each function takes one and returns the next.  Pages are shared between them and written in
place, but a call only writes slots that are free in the cache that it is given.  The cache given therefore stays valid (a step
that turns out wrong is undone by going on from the earlier value) until another call writes pages.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .. import _cabi
from ..backend import resolve_backend
from .attention import default_scale

__all__ = ["PagedCache", "paged_cache", "cache_append", "cache_fork", "cache_free", "cache_compact", "decode_attention"]


class PagedCache(NamedTuple):
    """Pages of ``k`` and ``v``, ``(pages, key heads, page size, head dim)``, and the int32 arrays that describe their use."""

    k_pages: torch.Tensor
    v_pages: torch.Tensor
    table: torch.Tensor         #: (sequences, width): the pages of each sequence in order
    lengths: torch.Tensor       #: (sequences,): tokens of each sequence
    free_pages: torch.Tensor    #: (pages,): of which free_range[0] .. free_range[1] are free, in the order of their use
    free_range: torch.Tensor    #: (2,)
    shortfall: torch.Tensor     #: (1,): tokens that the last call had no page for and dropped


def paged_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, *, sequences: int, max_length: int,
                dtype: torch.dtype = torch.bfloat16, device="cuda") -> PagedCache:
    """An empty cache for ``sequences`` sequences of up to ``max_length`` tokens."""
    for name, value in dict(pages=pages, page_size=page_size, kv_heads=kv_heads, head_dim=head_dim, max_length=max_length).items():
        if value < 1:
            raise ValueError(f"paged_cache: {name} must be positive; got {value}")
    shape = (pages, kv_heads, page_size, head_dim)
    ints = dict(dtype=torch.int32, device=device)
    return PagedCache(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device),
                      torch.full((sequences, -(-max_length // page_size)), -1, **ints), torch.zeros(sequences, **ints),
                      torch.arange(pages, **ints), torch.tensor([0, pages], **ints), torch.zeros(1, **ints))


def cache_append(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, *, backend: str = "auto") -> PagedCache:
    """The cache with tokens ``offsets[i] .. offsets[i + 1]`` of ``k`` and ``v`` ``(tokens, key heads, head dim)`` behind those
    of sequence ``i``; ``offsets`` is int32 ``(sequences + 1,)``.  New pages go to the sequences in order.  Tokens for which
    there is no page (or no room in the table) are dropped from the end of a sequence and counted in ``shortfall``, as are those
    that offsets name beyond ``k`` and ``v``; offsets that descend store nothing.  The cache holds values: no gradient flows back
    through it."""
    resolve_backend(backend)
    lengths, free_range, shortfall = _cabi.torch_ops().cache_append(*cache[:6], k, v, offsets)
    return cache._replace(lengths=lengths, free_range=free_range, shortfall=shortfall)


def cache_fork(cache: PagedCache, parents: torch.Tensor, *, backend: str = "auto") -> PagedCache:
    """The cache whose sequence ``i`` is a copy of sequence ``parents[i]`` (int32; any number of them; a negative one leaves
    the row empty).  Full pages are shared; the page that is still being filled is copied for every child but the first.  Pages
    that no sequence reaches any more are free; the list of free pages is then in ascending order."""
    resolve_backend(backend)
    return PagedCache(*cache[:2], *_cabi.torch_ops().cache_fork(*cache[:6], parents, False))


def cache_free(cache: PagedCache, finished: torch.Tensor, *, backend: str = "auto") -> PagedCache:
    """The cache without the sequences that ``finished`` (bool, ``(sequences,)``) names: their rows are empty."""
    resolve_backend(backend)
    return PagedCache(*cache[:2], *_cabi.torch_ops().cache_fork(*cache[:6], finished, True))


def cache_compact(cache: PagedCache, *, backend: str = "auto") -> PagedCache:
    """The cache with its live pages at the front of the pool: those behind move to the lowest free places, in order."""
    resolve_backend(backend)
    table, free_pages, free_range, shortfall = _cabi.torch_ops().cache_compact(*cache[:6])
    return cache._replace(table=table, free_pages=free_pages, free_range=free_range, shortfall=shortfall)


def decode_attention(q: torch.Tensor, cache: PagedCache, *, scale: Optional[float] = None, backend: str = "auto") -> torch.Tensor:
    """Attention of one query token per sequence, ``q`` ``(sequences, heads, head dim)``, over the sequence's tokens in the
    cache (the new token's own among them, once it has been appended).  Query head ``h`` reads key head
    ``h // (heads // key heads)``; an empty sequence gives zeros.  Not differentiable."""
    resolve_backend(backend)
    return _cabi.torch_ops().decode_attention(q, *cache[:4], default_scale(q.shape[-1]) if scale is None else float(scale))
