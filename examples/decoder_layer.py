"""The attention layer of a small decoder, trained on packed documents and then served from a paged cache.

    python -m examples.decoder_layer

Training runs ``rotary_embedding`` and ``packed_attention`` over documents of unequal length that lie one after the other.
Serving takes prompts in the same way, stores their keys and values with ``cache_append``, and generates a token per sequence and
step with ``decode_attention``; in between beams are chosen anew (``cache_fork``), finished ones leave (``cache_free``) and the
pool is packed (``cache_compact``).  No call of it waits for the GPU.
"""
from __future__ import annotations

import torch

from nitrix_b200.nn import (cache_append, cache_compact, cache_fork, cache_free, decode_attention, packed_attention, paged_cache,
                            rotary_embedding, rotary_frequencies)


class AttentionLayer:
    """Grouped-query attention with rotary positions: ``heads`` query heads on ``kv_heads`` key heads."""

    def __init__(self, width=256, heads=8, kv_heads=2, head_dim=64, dtype=torch.bfloat16, device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        rows = (heads + 2 * kv_heads) * head_dim
        self.w_in = (torch.randn(rows, width, generator=g, device=device) * width ** -0.5).to(dtype).requires_grad_(True)
        self.w_out = (torch.randn(width, heads * head_dim, generator=g, device=device) * (heads * head_dim) ** -0.5).to(dtype).requires_grad_(True)
        self.frequencies = rotary_frequencies((head_dim // 2,), device=device)

    def project(self, x, positions):
        """Queries and keys at their positions, and values, of tokens ``x`` (tokens, width)."""
        qkv = (x @ self.w_in.T).view(x.shape[0], -1, self.head_dim)
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=1)
        q, k = rotary_embedding(q, k, positions, self.frequencies)
        return q, k, v

    def packed(self, x, positions, offsets, cache=None):
        """All tokens of packed sequences at once; into ``cache`` as well, where there is one."""
        q, k, v = self.project(x, positions)
        if cache is not None:
            cache = cache_append(cache, k, v, offsets)
        out = packed_attention(q, k, v, offsets).flatten(1) @ self.w_out.T
        return out if cache is None else (out, cache)

    def step(self, x, cache):
        """One new token of every sequence, ``x`` (sequences, width)."""
        q, k, v = self.project(x, cache.lengths)
        each = torch.arange(x.shape[0] + 1, dtype=torch.int32, device=x.device)
        cache = cache_append(cache, k, v, each)
        return decode_attention(q, cache).flatten(1) @ self.w_out.T, cache


def pack(lengths, device="cuda"):
    """Offsets, and every token's position in its sequence."""
    offsets = torch.tensor([0, *lengths]).cumsum(0).int()
    positions = torch.cat([torch.arange(n) for n in lengths]).int()
    return offsets.to(device), positions.to(device)


def train(layer, lengths, steps=20, rate=8.0, seed=1):
    """Least squares towards random targets; the losses."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    offsets, positions = pack(lengths)
    width = layer.w_in.shape[1]
    x, target = (torch.randn(sum(lengths), width, generator=g, device="cuda").to(layer.w_in.dtype) for _ in range(2))
    losses = []
    for _ in range(steps):
        loss = (layer.packed(x, positions, offsets).float() - 0.1 * target.float()).square().mean()
        grads = torch.autograd.grad(loss, [layer.w_in, layer.w_out])
        with torch.no_grad():
            for w, grad in zip((layer.w_in, layer.w_out), grads):
                w -= rate * grad
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


@torch.no_grad()
def serve(layer, prompts, beams=2, steps=8):
    """Outputs of the prompts' last tokens and of every generated one, the cache, and the tokens that were fed (for a check).

    ``prompts``: a (length, width) tensor each.  A generated token's output, normalised, is the next token."""
    lengths = [p.shape[0] for p in prompts]
    offsets, positions = pack(lengths)
    cache = paged_cache(256, 16, layer.kv_heads, layer.head_dim, sequences=len(prompts), max_length=512, dtype=prompts[0].dtype)
    out, cache = layer.packed(torch.cat(prompts), positions, offsets, cache)
    last = out[offsets[1:].long() - 1]
    # every prompt is continued by several beams, which share its pages
    parents = torch.arange(len(prompts), device="cuda").repeat_interleave(beams).int()
    cache, last = cache_fork(cache, parents), last[parents.long()]
    fed, outputs = [], [last]
    for i in range(steps):
        # (beams of one prompt would all go the same way: each hears another tone)
        token = last / last.float().norm(dim=1, keepdim=True) * last.shape[1] ** 0.5
        token = (token + 0.1 * torch.arange(token.shape[0], device="cuda")[:, None]).to(last.dtype)
        last, cache = layer.step(token, cache)
        fed.append(token)
        outputs.append(last)
    finished = torch.arange(last.shape[0], device="cuda") % 3 == 2
    return outputs, fed, cache_compact(cache_free(cache, finished)), cache


if __name__ == "__main__":
    layer = AttentionLayer()
    losses = train(layer, [300, 17, 128, 1, 555])
    print("loss", " ".join(f"{x:.4f}" for x in losses[::5]))
    prompts = [torch.randn(n, 256, device="cuda").bfloat16() for n in (40, 7, 100)]
    outputs, _, packed, before = serve(layer, prompts)
    print("sequences", before.lengths.tolist(), "pages free", int(before.free_range[1] - before.free_range[0]))
    print("after three have finished", packed.lengths.tolist(), "pages free", int(packed.free_range[1] - packed.free_range[0]))
