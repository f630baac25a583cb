"""64-bit restatements of the operators of a decoder's attention layer -- TEST INFRASTRUCTURE ONLY.

Written from the formulas, on torch tensors of any device; the cache's bookkeeping is a model in plain Python lists.
``packed`` and ``decode`` return beside each value the sums that bound what rounding can do to it: a relative error ``u`` in the
probabilities and their gradients, and in the result, changes an entry by no more than ``u`` times the second tensor.
"""
from __future__ import annotations

import math

import numpy as np
import torch


def rotary(x, positions, frequencies, sections, interleaved=False, inverse=False):
    """``x`` (..., heads, D), ``positions`` (..., axes)."""
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    pairs = len(axis)
    # (the phases of far positions have more than 53 bits: formed and reduced in the host's long double)
    turn = np.longdouble("6.283185307179586476925286766559005768")
    phase = positions[..., axis].cpu().numpy().astype(np.longdouble) * frequencies.cpu().numpy().astype(np.longdouble)
    phase = torch.from_numpy((phase - np.rint(phase / turn) * turn).astype(np.float64)).to(x.device)
    cos, sin = torch.cos(phase)[..., None, :], torch.sin(phase)[..., None, :]
    if inverse:
        sin = -sin
    y = x.double().clone()
    first = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
    second = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
    a, b = x.double()[..., first], x.double()[..., second]
    y[..., first], y[..., second] = a * cos - b * sin, a * sin + b * cos
    return y


def _softmax(scores, seen):
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top)), torch.zeros_like(scores))
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, p / total, torch.zeros_like(p))


def packed(q, k, v, lengths_q, lengths_k, scale, causal, dout=None):
    """``{name: (value, bound)}`` of out and, with ``dout``, dq, dk, dv."""
    H, Hk = q.shape[1], k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    names = {"out": q} if dout is None else {"out": q, "dq": q, "dk": k, "dv": v}
    res = {n: (torch.zeros_like(t), torch.zeros_like(t)) for n, t in names.items()}
    sq = sk = 0
    for lq, lk in zip(lengths_q, lengths_k):
        rows, keys = slice(sq, sq + lq), slice(sk, sk + lk)
        sq, sk = sq + lq, sk + lk
        if lq == 0 or lk == 0:
            continue
        seen = torch.ones(lq, lk, dtype=torch.bool, device=q.device)
        if causal:
            seen = torch.arange(lk, device=q.device)[None] <= torch.arange(lq, device=q.device)[:, None] + lk - lq
        for h in range(H):
            g = h * Hk // H
            p = _softmax(scale * q[rows, h] @ k[keys, g].T, seen)
            o = p @ v[keys, g]
            res["out"][0][rows, h] = o
            res["out"][1][rows, h] = p @ v[keys, g].abs() + o.abs()
            if dout is None:
                continue
            do = dout[rows, h].double()
            ds = p * (do @ v[keys, g].T - (do * o).sum(-1, keepdim=True))
            ds_err = ds.abs() + p * (do * o).abs().sum(-1, keepdim=True)
            res["dq"][0][rows, h] = scale * ds @ k[keys, g]
            res["dq"][1][rows, h] = abs(scale) * ds_err @ k[keys, g].abs() + (scale * ds @ k[keys, g]).abs()
            for name, w, w_err, x in (("dk", scale * ds, abs(scale) * ds_err, q[rows, h]), ("dv", p, p, do)):
                res[name][0][keys, g] += w.T @ x
                res[name][1][keys, g] += w_err.T @ x.abs()
    if dout is not None:
        for name in ("dk", "dv"):
            res[name][1].add_(res[name][0].abs())
    return res


def decode(q, k_pages, v_pages, table, lengths, scale):
    """(value, bound) of the attention of one token per sequence."""
    H, Hk, page = q.shape[1], k_pages.shape[1], k_pages.shape[2]
    out, bound = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    for i, length in enumerate(lengths):
        if length == 0:
            continue
        at = torch.arange(length, device=q.device)
        pages, slots = table[i].long()[at // page], at % page
        for h in range(H):
            g = h * Hk // H
            p = torch.softmax(scale * k_pages[pages, g, slots].double() @ q[i, h].double(), 0)
            v = v_pages[pages, g, slots].double()
            out[i, h] = p @ v
            bound[i, h] = p @ v.abs() + (p @ v).abs()
    return out, bound


class CacheModel:
    """A paged cache of one head whose tokens are plain values; rows of page numbers, a free list."""

    def __init__(self, pages, page_size, sequences, width):
        self.pages, self.page_size, self.width = pages, page_size, width
        self.slots = [[None] * page_size for _ in range(pages)]
        self.table = [[] for _ in range(sequences)]
        self.lengths = [0] * sequences
        self.free = list(range(pages))
        self.shortfall = 0

    def tokens(self, row):
        return [self.slots[self.table[row][t // self.page_size]][t % self.page_size] for t in range(self.lengths[row])]

    def append(self, new):
        """``new``: the tokens of each row."""
        self.shortfall = 0
        for row, tokens in enumerate(new):
            # (a row that wants more than it gets keeps what it got: the pages that are left)
            for token in tokens:
                if self.lengths[row] == len(self.table[row]) * self.page_size:
                    if not self.free or len(self.table[row]) == self.width:
                        self.shortfall += 1
                        continue
                    self.table[row].append(self.free.pop(0))
                at = self.lengths[row]
                self.slots[self.table[row][at // self.page_size]][at % self.page_size] = token
                self.lengths[row] += 1

    def _collect(self):
        live = {p for row in self.table for p in row}
        self.free = [p for p in range(self.pages) if p not in live]

    def fork(self, parents):
        self.shortfall = 0
        table, lengths, taken = [], [], set()
        for parent in parents:
            if not 0 <= parent < len(self.table):
                table.append([])
                lengths.append(0)
                continue
            row, length = list(self.table[parent]), self.lengths[parent]
            full, part = divmod(length, self.page_size)
            if part and parent in taken:
                if self.free:
                    page = self.free.pop(0)
                    self.slots[page][:part] = self.slots[row[full]][:part]
                    row[full] = page
                else:
                    self.shortfall += part
                    row, length = row[:full], full * self.page_size
            taken.add(parent)
            table.append(row)
            lengths.append(length)
        self.table, self.lengths = table, lengths
        self._collect()

    def compact(self):
        self._collect()
        live = sorted({p for row in self.table for p in row})
        moved = dict(zip([p for p in live if p >= len(live)], self.free))
        for src, dst in moved.items():
            self.slots[dst] = list(self.slots[src])
        self.table = [[moved.get(p, p) for p in row] for row in self.table]
        self.shortfall = 0
        self._collect()
