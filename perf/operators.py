"""Operators of a decoder's attention layer, as cases that a timing program can run one by one.

``rotary``   rotary positions of one or several axes, queries and keys together; forward, and forward with gradients
``append``   keys and values of new tokens into a paged cache: whole prompts, or one token per sequence
``fork``     the rows of a paged cache chosen anew (beams, finished sequences): forking, freeing, copying open pages
``compact``  the live pages of a cache moved to its front
``decode``   attention of one new token per sequence over the paged cache
``packed``   attention over packed sequences of unequal lengths with grouped heads; forward, and forward with gradients

``run`` computes them in elementary torch operations; with ``own`` set it calls this package's operators.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _rotary(name, *, dtype, tokens, H, Hk, D, sections, interleaved=False, train=False):
    """``sections``: rotated pairs per axis, as a text ("16,24,24"); twice their sum may be less than ``D``."""
    case = dict(op="rotary", dtype=dtype, tokens=tokens, H=H, Hk=Hk, D=D, sections=sections, interleaved=interleaved, train=train)
    return dict(name=name, **case) if name else case


def _append(name, *, dtype, n, held, new, Hk, D, page):
    """``n`` sequences that hold up to ``held`` tokens and get up to ``new`` each (exactly one where ``new`` is 1)."""
    case = dict(op="append", dtype=dtype, n=n, held=held, new=new, Hk=Hk, D=D, page=page)
    return dict(name=name, **case) if name else case


def _fork(name, *, dtype, n, held, Hk, D, page):
    case = dict(op="fork", dtype=dtype, n=n, held=held, Hk=Hk, D=D, page=page)
    return dict(name=name, **case) if name else case


def _compact(name, *, dtype, n, held, Hk, D, page):
    """A pool of twice the pages that ``n`` sequences of up to ``held`` tokens need, used at random."""
    case = dict(op="compact", dtype=dtype, n=n, held=held, Hk=Hk, D=D, page=page)
    return dict(name=name, **case) if name else case


def _decode(name, *, dtype, n, held, Hk, G, D, page):
    case = dict(op="decode", dtype=dtype, n=n, held=held, Hk=Hk, G=G, D=D, page=page)
    return dict(name=name, **case) if name else case


def _packed(name, *, dtype, n, longest, Hk, G, D, causal=True, train=False):
    case = dict(op="packed", dtype=dtype, n=n, longest=longest, Hk=Hk, G=G, D=D, causal=causal, train=train)
    return dict(name=name, **case) if name else case


def listed():
    return [
        # one new token of each of 64 sequences: the smallest call, where latency counts
        _rotary("rotary_token_f16", dtype="f16", tokens=64, H=32, Hk=8, D=128, sections="64"),
        # a training step over video tokens with (time, height, width) positions
        _rotary("rotary_video_train_bf16", dtype="bf16", tokens=16384, H=16, Hk=16, D=128, sections="16,24,24", train=True),
        # a batch of prompts of unequal length enters an empty cache
        _append("append_prompts_bf16", dtype="bf16", n=16, held=0, new=4096, Hk=8, D=128, page=16),
        # one step of generation: a token per sequence
        _append("append_token_f16", dtype="f16", n=256, held=2048, new=1, Hk=4, D=64, page=16),
        # a beam search chooses its survivors
        _fork("fork_beams_f32", dtype="f32", n=64, held=1000, Hk=8, D=64, page=64),
        # a half-empty, fragmented pool is packed
        _compact("compact_bf16", dtype="bf16", n=64, held=2048, Hk=8, D=128, page=16),
        # a single short conversation
        _decode("decode_one_f32", dtype="f32", n=1, held=1000, Hk=4, G=2, D=64, page=16),
        # a served batch of unequal lengths, some slots empty
        _decode("decode_batch_bf16", dtype="bf16", n=64, held=8192, Hk=8, G=4, D=128, page=16),
        # few very long contexts: the split over the length is what fills the GPU
        _decode("decode_long_f16", dtype="f16", n=4, held=131072, Hk=8, G=8, D=128, page=64),
        # a handful of short prompts: a small call
        _packed("packed_short_f16", dtype="f16", n=12, longest=300, Hk=2, G=4, D=64),
        # long prompts of unequal length; the largest in operations
        _packed("packed_long_bf16", dtype="bf16", n=8, longest=16384, Hk=8, G=4, D=128),
        # a training step over packed documents
        _packed("packed_train_bf16", dtype="bf16", n=16, longest=4096, Hk=4, G=4, D=128, train=True),
    ]


# ---- further cases of the same ranges ------------------------------------------------------------------------------
def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "append", "fork", "compact", "decode", "decode", "decode", "packed", "packed",
                     "packed", "packed"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    Hk, G, D = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8, 16]), rng.choice([64, 128])
    page = rng.choice([16, 32, 64, 128])
    if op == "rotary":
        pairs = D // 2 if rng.random() < 0.7 else D // 4
        axes = rng.choice([1, 1, 2, 3])
        cut = sorted(rng.sample(range(1, pairs), axes - 1))
        sections = ",".join(str(b - a) for a, b in zip([0, *cut], [*cut, pairs]))
        tokens, train = _log_int(rng, 1, 16384), rng.random() < 0.5
        while tokens * Hk * (G + 1) * D * _BYTES[dtype] > 16384 * 32 * 128 * 2:
            tokens = (tokens + 1) // 2
        return _rotary(None, dtype=dtype, tokens=tokens, H=Hk * G, Hk=Hk, D=D, sections=sections,
                       interleaved=rng.random() < 0.4, train=train)
    if op == "append":
        n, new = _log_int(rng, 1, 256), 1 if rng.random() < 0.5 else _log_int(rng, 2, 4096)
        held = _log_int(rng, 1, 2048)
        while n * (held + new) * Hk * D * _BYTES[dtype] > 1 << 27:
            n, held, new = (n + 1) // 2, (held + 1) // 2, (new + 1) // 2
        return _append(None, dtype=dtype, n=n, held=held, new=new, Hk=Hk, D=D, page=page)
    if op in ("fork", "compact"):
        n, held = _log_int(rng, 1, 128), _log_int(rng, 1, 4096)
        while n * held * Hk * D * _BYTES[dtype] > 1 << 28:
            n, held = (n + 1) // 2, (held + 1) // 2
        return (_fork if op == "fork" else _compact)(None, dtype=dtype, n=n, held=held, Hk=Hk, D=D, page=page)
    if op == "decode":
        n, held = _log_int(rng, 1, 256), _log_int(rng, 1, 131072)
        while n * held * Hk * D * _BYTES[dtype] > 1 << 29:
            n, held = (n + 1) // 2, (held + 1) // 2
        return _decode(None, dtype=dtype, n=n, held=held, Hk=Hk, G=G, D=D, page=page)
    n, longest, train = _log_int(rng, 1, 64), _log_int(rng, 1, 2048 if dtype == "f32" else 16384), rng.random() < 0.5
    limit = 2e8 if dtype == "f32" else 2e9      # (query head, query, key) triples, below those of the listed cases
    while n * longest * longest * Hk * G > limit:
        n, longest = (n + 1) // 2, max(1, int(longest * 0.7))
    return _packed(None, dtype=dtype, n=n, longest=longest, Hk=Hk, G=G, D=D, causal=rng.random() < 0.8, train=train)


# ---- inputs ------------------------------------------------------------------------------------------------------
def _lengths(n, longest):
    """Lengths of a batch: evenly spaced up to ``longest`` with odd ones among them; eight or more hold an empty one and
    one of a single token."""
    out = [max(1, round(longest * (i + 1) / n) - (7 * i % 13 if i + 1 < n else 0)) for i in range(n)]
    if n >= 8:
        out[0], out[1] = 0, 1
    return out


def _dealt(lengths, seed):
    """The lengths in an order that the seed decides."""
    order = torch.randperm(len(lengths), generator=torch.Generator().manual_seed(seed)).tolist()
    return [lengths[i] for i in order]


def _offsets(lengths):
    return torch.tensor([0, *lengths], dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def _randn(g, shape, dtype, std=1.0):
    out = torch.empty(shape, device="cuda", dtype=dtype)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 28):           # bounded fp32 temporaries
        part = flat[i:i + (1 << 28)]
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * std)
    return out


def _frequencies(sections):
    """Every axis has a ladder of its own: 10000 ^ (-j / pairs of the axis)."""
    rows = [torch.pow(torch.tensor(10000.0, dtype=torch.float64), -torch.arange(s, dtype=torch.float64) / s) for s in sections]
    return torch.cat(rows).float().cuda()


def _pages_of(case):
    """Pages that the held tokens take, and the pool's size."""
    page, n = case["page"], case["n"]
    held = [-(-x // page) for x in _lengths(n, case["held"])] if case["held"] else [0] * n
    live = sum(held)
    if case["op"] == "append":
        return held, live + sum(-(-x // page) + 1 for x in _new_lengths(case)) + 8
    if case["op"] == "fork":
        return held, live + n + 8
    if case["op"] == "compact":
        return held, 2 * live + 8
    return held, live + 8


def _new_lengths(case):
    return [1] * case["n"] if case["new"] == 1 else _lengths(case["n"], case["new"])


def _cache(case, g, seed):
    """A pool in use: pages in random order, stale values where no sequence has written yet."""
    page, n = case["page"], case["n"]
    _, pool = _pages_of(case)
    lengths = _dealt(_lengths(n, case["held"]) if case["held"] else [0] * n, seed)
    most = max(lengths) + (max(_new_lengths(case)) if case["op"] == "append" else 0)
    width = max(1, -(-most // page))
    order = torch.randperm(pool, generator=g, device="cuda").int()
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, length in enumerate(lengths):
        need = -(-length // page)
        table[i, :need] = order[at:at + need]
        at += need
    free = torch.full((pool,), -1, dtype=torch.int32, device="cuda")
    free[:pool - at] = order[at:]
    shape = (pool, case["Hk"], page, case["D"])
    dt = _DTYPES[case["dtype"]]
    return dict(k_pages=_randn(g, shape, dt), v_pages=_randn(g, shape, dt), table=table,
                lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), free_pages=free,
                free_range=torch.tensor([0, pool - at], dtype=torch.int32, device="cuda"),
                shortfall=torch.zeros(1, dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, op = _DTYPES[case["dtype"]], case["op"]
    state = dict(op=op)
    if op == "rotary":
        tokens, D = case["tokens"], case["D"]
        sections = tuple(int(s) for s in case["sections"].split(","))
        state.update(q=_randn(g, (tokens, case["H"], D), dt), k=_randn(g, (tokens, case["Hk"], D), dt), sections=sections,
                     frequencies=_frequencies(sections), interleaved=case["interleaved"], grads=None)
        if len(sections) == 1:      # a long context, continued somewhere
            start = torch.randint(0, 131072, (1,), generator=g, device="cuda")
            state["positions"] = (start + torch.arange(tokens, device="cuda"))[:, None].int()
        else:                       # frames of up to 24 x 32 patches
            t = torch.arange(tokens, device="cuda") + torch.randint(0, 4096, (1,), generator=g, device="cuda")
            state["positions"] = torch.stack([t // 768, t // 32 % 24, t % 32][:len(sections)], dim=1).int()
        if case["train"]:
            state["grads"] = (_randn(g, (tokens, case["H"], D), dt), _randn(g, (tokens, case["Hk"], D), dt))
        return state
    if op == "packed":
        lengths = _dealt(_lengths(case["n"], case["longest"]), seed)
        total, Hk, G, D = sum(lengths), case["Hk"], case["G"], case["D"]
        state.update(q=_randn(g, (total, Hk * G, D), dt), k=_randn(g, (total, Hk, D), dt), v=_randn(g, (total, Hk, D), dt),
                     offsets=_offsets(lengths), lengths=lengths, causal=case["causal"], dout=None)
        if case["train"]:
            state["dout"] = _randn(g, (total, Hk * G, D), dt)
        return state
    state["cache"] = _cache(case, g, seed)
    if op == "append":
        new = _dealt(_new_lengths(case), seed + 1)
        state.update(k=_randn(g, (sum(new), case["Hk"], case["D"]), dt), v=_randn(g, (sum(new), case["Hk"], case["D"]), dt),
                     offsets=_offsets(new))
    elif op == "fork":
        # four beams per prompt: survivors are drawn from the four, every seventh row has finished
        n = case["n"]
        rows = torch.arange(n, device="cuda")
        pick = torch.randint(0, 4, (n,), generator=g, device="cuda")
        parents = torch.clamp(rows // 4 * 4 + pick, max=n - 1)
        state["parents"] = torch.where(rows % 7 == 6, torch.full_like(parents, -1), parents).int()
    elif op == "decode":
        state["q"] = _randn(g, (case["n"], case["Hk"] * case["G"], case["D"]), dt)
    return state


# ---- one pass ------------------------------------------------------------------------------------------------------
_CACHE_FIELDS = ("k_pages", "v_pages", "table", "lengths", "free_pages", "free_range", "shortfall")


def _run_own(state):
    from nitrix_b200 import nn

    op = state["op"]
    if op == "rotary":
        q, k = state["q"], state["k"]
        args = dict(sections=state["sections"], interleaved=state["interleaved"])
        if state["grads"] is None:
            return list(nn.rotary_embedding(q, k, state["positions"], state["frequencies"], **args))
        q.requires_grad_(True), k.requires_grad_(True)
        out = nn.rotary_embedding(q, k, state["positions"], state["frequencies"], **args)
        return [out[0].detach(), out[1].detach(), *torch.autograd.grad(out, [q, k], state["grads"])]
    if op == "packed":
        leaves = [state["q"], state["k"], state["v"]]
        if state["dout"] is not None:
            for t in leaves:
                t.requires_grad_(True)
        out = nn.packed_attention(*leaves, state["offsets"], causal=state["causal"])
        if state["dout"] is None:
            return [out]
        return [out.detach(), *torch.autograd.grad(out, leaves, state["dout"])]
    cache = nn.PagedCache(**state["cache"])
    if op == "decode":
        return [nn.decode_attention(state["q"], cache)]
    if op == "append":
        cache = nn.cache_append(cache, state["k"], state["v"], state["offsets"])
    elif op == "fork":
        cache = nn.cache_fork(cache, state["parents"])
    else:
        cache = nn.cache_compact(cache)
    return [getattr(cache, name) for name in _CACHE_FIELDS]


@torch.no_grad()
def run(state):
    if own:
        with torch.enable_grad():
            return _run_own(state)
    return {"rotary": _plain_rotary, "append": _plain_append, "fork": _plain_fork, "compact": _plain_compact,
            "decode": _plain_decode, "packed": _plain_packed}[state["op"]](state)


def _plain_rotary(state):
    axis = torch.cat([torch.full((s,), a) for a, s in enumerate(state["sections"])]).to("cuda")
    # the phases of far positions need more than 32 bits (131072 * 2^-24 is an error of 0.008); all else is held in 32
    phase = state["positions"].double()[:, axis] * state["frequencies"].double()
    cos, sin = torch.cos(phase).float()[:, None], torch.sin(phase).float()[:, None]
    pairs = cos.shape[-1]

    def rotate(x, sin):
        y = x.float()
        if state["interleaved"]:
            a, b = y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2]
            turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
        else:
            a, b = y[..., :pairs], y[..., pairs:2 * pairs]
            turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
        return torch.cat([turned, y[..., 2 * pairs:]], dim=-1).to(x.dtype)

    out = [rotate(state["q"], sin), rotate(state["k"], sin)]
    if state["grads"] is not None:
        out += [rotate(g, -sin) for g in state["grads"]]
    return out


def _plain_append(state):
    c = state["cache"]
    page, width, pool = c["k_pages"].shape[2], c["table"].shape[1], c["k_pages"].shape[0]
    offsets, held = state["offsets"].long(), c["lengths"].long()
    begin, end = c["free_range"].long().unbind()
    want = held + offsets[1:] - offsets[:-1]
    have = (held + page - 1) // page
    need = torch.clamp(torch.clamp((want + page - 1) // page, max=width) - have, min=0)
    before = need.cumsum(0) - need
    got = torch.minimum(torch.clamp(end - begin - before, min=0), need)
    lengths = torch.minimum(want, (have + got) * page)
    column = torch.arange(width, device="cuda")[None]
    fresh = c["free_pages"].long()[torch.clamp(begin + before[:, None] + column - have[:, None], 0, pool - 1)]
    is_new = (column >= have[:, None]) & (column < (have + got)[:, None])
    table = torch.where(is_new, fresh, c["table"].long())
    c["table"].copy_(table)
    t = torch.arange(state["k"].shape[0], device="cuda")
    row = torch.searchsorted(offsets[1:].contiguous(), t, right=True)
    at = held[row] + t - offsets[row]
    target = table[row, torch.clamp(at // page, max=width - 1)]
    c["k_pages"][target, :, at % page] = state["k"]      # (the pools of these cases hold every token)
    c["v_pages"][target, :, at % page] = state["v"]
    free_range = torch.stack([begin + got.sum(), end]).int()
    return [c["k_pages"], c["v_pages"], c["table"], lengths.int(), c["free_pages"], free_range, (want - lengths).sum().int()[None]]


def _plain_live(table, lengths, page, pool):
    """Which pages the rows reach, and the pages that none does in ascending order, -1 behind them."""
    column = torch.arange(table.shape[1], device="cuda")[None]
    reached = torch.where(column < (lengths[:, None] + page - 1) // page, table, torch.full_like(table, pool))
    live = torch.zeros(pool + 1, dtype=torch.bool, device="cuda")
    live[reached.flatten()] = True
    live = live[:pool]
    rank = (~live).cumsum(0) - 1
    free = torch.full((pool + 1,), -1, dtype=torch.int64, device="cuda")
    free[torch.where(live, torch.full_like(rank, pool), rank)] = torch.where(live, torch.full_like(rank, -1),
                                                                             torch.arange(pool, device="cuda"))
    return live, free[:pool]


def _plain_fork(state):
    c = state["cache"]
    page, width, pool = c["k_pages"].shape[2], c["table"].shape[1], c["k_pages"].shape[0]
    parents = state["parents"].long()
    begin, end = c["free_range"].long().unbind()
    there = parents >= 0
    source = torch.clamp(parents, min=0)
    held = torch.where(there, c["lengths"].long()[source], torch.zeros_like(parents))
    rows = torch.arange(parents.shape[0], device="cuda")
    first = ~((parents[:, None] == parents[None]) & (rows[None] < rows[:, None])).any(1)
    full, part = held // page, held % page
    copies = (part > 0) & ~first
    rank = copies.long().cumsum(0) - copies.long()
    served = copies & (rank < end - begin)
    lengths = torch.where(copies & ~served, full * page, held)
    fresh = c["free_pages"].long()[torch.clamp(begin + rank, 0, pool - 1)]
    column = torch.arange(width, device="cuda")[None]
    table = torch.where(column < ((lengths + page - 1) // page)[:, None], c["table"].long()[source], torch.full((1,), -1, device="cuda"))
    table = torch.where(served[:, None] & (column == full[:, None]), fresh[:, None], table)
    # one row after the other: a row that copies nothing writes a page onto itself
    old = torch.clamp(c["table"].long()[source].gather(1, torch.clamp(full, max=width - 1)[:, None]), min=0)
    new = torch.where(served[:, None], fresh[:, None], old)
    kept = (torch.arange(page, device="cuda")[None] < part[:, None])[:, None, :, None]
    for pages in (c["k_pages"], c["v_pages"]):
        for i in range(parents.shape[0]):
            pages[new[i]] = torch.where(kept[i], pages[old[i]], pages[new[i]])
    _, free = _plain_live(table, lengths, page, pool)
    free_range = torch.stack([torch.zeros_like(begin), (free >= 0).sum()]).int()
    return [c["k_pages"], c["v_pages"], table.int(), lengths.int(), free.int(), free_range, (held - lengths).sum().int()[None]]


def _plain_compact(state):
    c = state["cache"]
    page, width, pool = c["k_pages"].shape[2], c["table"].shape[1], c["k_pages"].shape[0]
    lengths, table = c["lengths"].long(), c["table"].long()
    live, free = _plain_live(table, lengths, page, pool)
    n_live = live.sum()
    index = torch.arange(pool, device="cuda")
    moves = live & (index >= n_live)
    to = torch.where(moves, free[torch.clamp(moves.long().cumsum(0) - 1, min=0)], index)
    origin = torch.cat([index, index[:1]])
    origin[torch.where(moves, to, torch.full_like(to, pool))] = index
    for pages in (c["k_pages"], c["v_pages"]):
        pages.copy_(pages[origin[:pool]])
    column = torch.arange(width, device="cuda")[None]
    table = torch.where(column < ((lengths + page - 1) // page)[:, None], to[torch.clamp(table, min=0)], torch.full((1,), -1, device="cuda"))
    free = torch.where(index < pool - n_live, index + n_live, torch.full_like(index, -1))
    free_range = torch.stack([torch.zeros_like(n_live), pool - n_live]).int()
    return [c["k_pages"], c["v_pages"], table.int(), lengths.int(), free.int(), free_range, torch.zeros(1, dtype=torch.int32, device="cuda")]


def _plain_decode(state):
    c, q = state["cache"], state["q"]
    (n, H, D), (_, Hk, page, _) = q.shape, c["k_pages"].shape
    out = torch.empty_like(q)
    width = c["table"].shape[1]
    at = torch.arange(width * page, device="cuda")
    for i in range(n):
        row = torch.clamp(c["table"][i].long(), min=0)
        keep = at < c["lengths"][i]
        k = c["k_pages"][row].transpose(0, 1).reshape(Hk, width * page, D).float()
        v = c["v_pages"][row].transpose(0, 1).reshape(Hk, width * page, D).float()
        s = (q[i].float().view(Hk, H // Hk, D) @ k.transpose(1, 2)) / math.sqrt(D)
        s = torch.where(keep, s, torch.full((), -math.inf, device="cuda"))
        p = torch.where(keep, torch.exp(s - s.amax(-1, keepdim=True)), torch.zeros((), device="cuda"))
        total = p.sum(-1, keepdim=True)
        o = (p @ torch.where(keep[:, None], v, torch.zeros((), device="cuda"))) / torch.where(total > 0, total, torch.ones_like(total))
        out[i] = o.reshape(H, D).to(q.dtype)
    return [out]


def _plain_packed(state):
    q, k, v, dout = state["q"], state["k"], state["v"], state["dout"]
    H, Hk, D = q.shape[1], k.shape[1], q.shape[2]
    G, scale = H // Hk, 1.0 / math.sqrt(D)
    out = torch.empty_like(q)
    grads = [] if dout is None else [torch.empty_like(t) for t in (q, k, v)]
    start = 0
    for length in state["lengths"]:
        s = slice(start, start + length)
        start += length
        if length == 0:
            continue
        later = torch.arange(length, device="cuda")[None] > torch.arange(length, device="cuda")[:, None]
        for h in range(Hk):
            heads = slice(h * G, (h + 1) * G)
            qh, kh, vh = q[s, heads].transpose(0, 1).float(), k[s, h].float(), v[s, h].float()
            p = (qh @ kh.t()) * scale
            if state["causal"]:
                p.masked_fill_(later, -math.inf)
            p.sub_(p.amax(-1, keepdim=True)).exp_()
            p.div_(p.sum(-1, keepdim=True))
            o = p @ vh
            out[s, heads] = o.transpose(0, 1).to(q.dtype)
            if dout is not None:
                do = dout[s, heads].transpose(0, 1).float()
                grads[2][s, h] = (p.transpose(1, 2) @ do).sum(0).to(v.dtype)
                ds = p * (do @ vh.t() - (do * o).sum(-1, keepdim=True))
                grads[0][s, heads] = ((ds @ kh) * scale).transpose(0, 1).to(q.dtype)
                grads[1][s, h] = ((ds.transpose(1, 2) @ qh).sum(0) * scale).to(k.dtype)
    return [out, *grads]


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def _pairs(lengths, causal):
    return sum(x * (x + 1) // 2 if causal else x * x for x in lengths)


def work(case):
    esz, op = _BYTES[case["dtype"]], case["op"]
    if op == "rotary":
        n = case["tokens"] * (case["H"] + case["Hk"]) * case["D"]
        axes = case["sections"].count(",") + 1
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * n * esz + 4 * axes * case["tokens"]), "flops": passes * 3 * n}
    if op == "packed":
        lengths, H, Hk, D = _lengths(case["n"], case["longest"]), case["Hk"] * case["G"], case["Hk"], case["D"]
        total, pairs = sum(lengths), _pairs(lengths, case["causal"]) * H
        q, kv = total * H * D * esz, total * Hk * D * esz
        if not case["train"]:
            return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * D}
        return {"bytes": 2 * q + 2 * kv + 4 * q + 4 * kv, "flops": 14 * pairs * D}
    page, row = case["page"], 2 * case["Hk"] * case["D"] * esz          # a token's key and value
    held = _lengths(case["n"], case["held"]) if case["held"] else [0] * case["n"]
    if op == "append":
        return {"bytes": 2 * sum(_new_lengths(case)) * row + 16 * case["n"], "flops": 0}
    _, pool = _pages_of(case)
    live = sum(-(-x // page) for x in held)
    if op == "fork":
        # of four beams about 4 (1 - 1 / e) have a child, the other rows copy half a page on average
        return {"bytes": int(0.3 * case["n"]) * page * row + 8 * live + 4 * pool, "flops": 0}
    if op == "compact":
        moved = live * (pool - live) // pool
        return {"bytes": 2 * moved * page * row + 8 * live + 4 * pool, "flops": 0}
    q = case["n"] * case["Hk"] * case["G"] * case["D"]
    return {"bytes": sum(held) * row + 2 * q * esz + 4 * live, "flops": 4 * sum(held) * case["Hk"] * case["G"] * case["D"]}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    """Computed numbers from their definitions in 64 bits; the cache's operators only move values and count."""
    op = case["op"]
    if op in ("append", "fork", "compact"):
        return None
    state = prepare(case, seed)
    with torch.enable_grad():
        return {"rotary": _exact_rotary, "decode": _exact_decode, "packed": _exact_packed}[op](state)


def _exact_rotary(state):
    """A pair is a complex number, turned by exp(i phase)."""
    bounds = torch.tensor(state["sections"]).cumsum(0)
    pairs = int(bounds[-1])
    axis = torch.bucketize(torch.arange(pairs), bounds, right=True).cuda()
    phase = torch.index_select(state["positions"].double(), 1, axis) * state["frequencies"].double()
    turn = torch.polar(torch.ones_like(phase), phase)[:, None]

    def rotate(x, turn):
        y = x.detach().double().clone()
        head = y[..., :2 * pairs]
        as_pairs = head.unflatten(-1, (pairs, 2)) if state["interleaved"] else head.unflatten(-1, (2, pairs)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(as_pairs.contiguous()) * turn)
        y[..., :2 * pairs] = (z if state["interleaved"] else z.transpose(-1, -2)).flatten(-2)
        return y

    out = [rotate(state["q"], turn), rotate(state["k"], turn)]
    if state["grads"] is not None:
        out += [rotate(g, turn.conj()) for g in state["grads"]]
    return out


def _exact_decode(state):
    c, q = state["cache"], state["q"]
    (n, H, D), (_, Hk, page, _) = q.shape, c["k_pages"].shape
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for i, length in enumerate(c["lengths"].tolist()):
        if length == 0:
            continue
        at = torch.arange(length, device="cuda")
        pages, slots = c["table"][i].long()[at // page], at % page
        for h in range(Hk):
            heads = slice(h * (H // Hk), (h + 1) * (H // Hk))
            logits = torch.einsum("gd,td->gt", q[i, heads].double(), c["k_pages"][pages, h, slots].double()) * D ** -0.5
            out[i, heads] = torch.einsum("gt,td->gd", torch.softmax(logits, dim=-1), c["v_pages"][pages, h, slots].double())
    return [out]


def _exact_packed(state):
    """Blocks of queries of one head, gradients by differentiation."""
    H, Hk, D = state["q"].shape[1], state["k"].shape[1], state["q"].shape[2]
    train = state["dout"] is not None
    q, k, v = (state[name].detach().double().requires_grad_(train) for name in ("q", "k", "v"))
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    grads = [torch.zeros_like(t) for t in (q, k, v)] if train else []
    start = 0
    for length in state["lengths"]:
        for h in range(H):
            for i in range(0, length, 4096):
                rows = slice(start + i, start + min(i + 4096, length))
                keys = slice(start, rows.stop if state["causal"] else start + length)
                leaves = [q[rows, h].detach(), k[keys, h * Hk // H].detach(), v[keys, h * Hk // H].detach()]
                for t in leaves:
                    t.requires_grad_(train)
                logits = torch.einsum("id,jd->ij", leaves[0], leaves[1]) * D ** -0.5
                if state["causal"]:
                    logits = logits.masked_fill(torch.ones_like(logits, dtype=torch.bool).triu(rows.start - start + 1), -math.inf)
                o = torch.softmax(logits, dim=-1) @ leaves[2]
                out[rows, h] = o.detach()
                if train:
                    for total, part, where in zip(grads, torch.autograd.grad(o, leaves, state["dout"][rows, h].double()),
                                                  ((rows, h), (keys, h * Hk // H), (keys, h * Hk // H))):
                        total[where] += part
        start += length
    return [out, *grads]
