"""Operators of a decoder layer in few bits, as cases that a timing program can run one by one.

``norm``     root-mean-square norm with the addition of the residual stream; forward, forward with gradients, or with an output
             in 8 bits (e4m3) and scales of rows or of groups of channels
``append``   keys and values of new tokens into a paged cache of 4 or 8 bits, and these tokens read back
``read``     all tokens of a cache of 4 or 8 bits as packed rows
``decode``   attention of one new token per sequence over a cache of 4 or 8 bits

``run`` computes them in elementary torch operations; with ``own`` set it calls this package's operators.

The cache.  A group is 32 elements of a head's row, with one fp16 step; a value is ``step * (code - 2^(bits - 1))``.  A row of
codes is ``(8, groups, bits / 2)`` bytes: of every group the elements ``4 j .. 4 j + 3`` lie together, the first in the lowest bits.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_EPS = 1e-6
_LEAST = 2.0 ** -100        # the largest value of a row counts as this much at least


def _norm(name, *, dtype, rows, C, mode, residual=True, weight=True, group=0):
    """``mode``: "forward", "train" or "eight" (``group`` channels share a scale, 0: a whole row)."""
    case = dict(op="norm", dtype=dtype, rows=rows, C=C, mode=mode, residual=residual, weight=weight, group=group)
    return dict(name=name, **case) if name else case


def _append(name, *, dtype, bits, n, held, new, Hk, D, page):
    """``n`` sequences that hold up to ``held`` tokens and get up to ``new`` each (exactly one where ``new`` is 1)."""
    case = dict(op="append", dtype=dtype, bits=bits, n=n, held=held, new=new, Hk=Hk, D=D, page=page)
    return dict(name=name, **case) if name else case


def _read(name, *, dtype, bits, n, held, Hk, D, page):
    case = dict(op="read", dtype=dtype, bits=bits, n=n, held=held, Hk=Hk, D=D, page=page)
    return dict(name=name, **case) if name else case


def _decode(name, *, dtype, bits, n, held, Hk, G, D, page):
    case = dict(op="decode", dtype=dtype, bits=bits, n=n, held=held, Hk=Hk, G=G, D=D, page=page)
    return dict(name=name, **case) if name else case


def listed():
    return [
        # one new token of each of 64 sequences before its attention: the smallest call, where latency counts
        _norm("norm_token_f16", dtype="f16", rows=64, C=4096, mode="forward"),
        # a training step over 16384 tokens
        _norm("norm_train_bf16", dtype="bf16", rows=16384, C=4096, mode="train"),
        # a long prompt before an 8-bit matrix product, a scale for every 128 channels
        _norm("norm_eight_bf16", dtype="bf16", rows=16384, C=8192, mode="eight", group=128),
        # odd rows and channels, fp32, with gradients
        _norm("norm_odd_f32", dtype="f32", rows=4099, C=1001, mode="train"),
        # a batch of prompts of unequal length enters an empty cache
        _append("append_prompts_4_bf16", dtype="bf16", bits=4, n=16, held=0, new=4096, Hk=8, D=128, page=16),
        # one step of generation: a token per sequence
        _append("append_token_8_f16", dtype="f16", bits=8, n=256, held=2048, new=1, Hk=4, D=64, page=16),
        # the contexts that the next chunks of their prompts attend to
        _read("read_contexts_4_bf16", dtype="bf16", bits=4, n=16, held=8192, Hk=8, D=128, page=16),
        # a single context in fp32
        _read("read_one_8_f32", dtype="f32", bits=8, n=1, held=1000, Hk=4, D=64, page=32),
        # a single short conversation
        _decode("decode_one_4_f32", dtype="f32", bits=4, n=1, held=1000, Hk=4, G=2, D=64, page=16),
        # a served batch of unequal lengths, some slots empty
        _decode("decode_batch_4_bf16", dtype="bf16", bits=4, n=64, held=8192, Hk=8, G=4, D=128, page=16),
        # the same in 8 bits, smaller heads
        _decode("decode_batch_8_bf16", dtype="bf16", bits=8, n=64, held=8192, Hk=8, G=5, D=64, page=64),
        # few very long contexts: the split over the length is what fills the GPU
        _decode("decode_long_4_f16", dtype="f16", bits=4, n=4, held=131072, Hk=8, G=8, D=128, page=64),
    ]


# ---- further cases of the same ranges ------------------------------------------------------------------------------
def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm", "append", "append", "read", "read", "decode", "decode", "decode", "decode"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "norm":
        mode = rng.choice(["forward", "train", "eight"])
        rows, C = _log_int(rng, 1, 16384), _log_int(rng, 16, 8192)
        if rng.random() < 0.7:
            C = max(64, C // 64 * 64)          # most models have round widths
        while rows * C * _BYTES[dtype] > 16384 * 4096 * 2:
            rows = (rows + 1) // 2
        group = rng.choice([0, 32, 64, 128]) if mode == "eight" else 0
        if group:
            C = max(group, C // group * group)
        return _norm(None, dtype=dtype, rows=rows, C=C, mode=mode, residual=rng.random() < 0.7, weight=rng.random() < 0.8, group=group)
    bits = rng.choice([4, 4, 8])
    Hk, G, D = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8, 16]), rng.choice([64, 128])
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        n, new = _log_int(rng, 1, 256), 1 if rng.random() < 0.5 else _log_int(rng, 2, 4096)
        held = _log_int(rng, 1, 2048)
        while n * (held + new) * Hk * D * _BYTES[dtype] > 1 << 27:
            n, held, new = (n + 1) // 2, (held + 1) // 2, (new + 1) // 2
        return _append(None, dtype=dtype, bits=bits, n=n, held=held, new=new, Hk=Hk, D=D, page=page)
    if op == "read":
        n, held = _log_int(rng, 1, 128), _log_int(rng, 1, 8192)
        while n * held * Hk * D * _BYTES[dtype] > 1 << 28:
            n, held = (n + 1) // 2, (held + 1) // 2
        return _read(None, dtype=dtype, bits=bits, n=n, held=held, Hk=Hk, D=D, page=page)
    n, held = _log_int(rng, 1, 256), _log_int(rng, 1, 131072)
    while n * held * Hk * D > 1 << 28 or n * held * Hk * G > 1 << 25:
        n, held = (n + 1) // 2, (held + 1) // 2
    return _decode(None, dtype=dtype, bits=bits, n=n, held=held, Hk=Hk, G=G, D=D, page=page)


# ---- inputs ------------------------------------------------------------------------------------------------------
def _lengths(n, longest):
    """Lengths of a batch: evenly spaced up to ``longest`` with odd ones among them; eight or more hold an empty one and
    one of a single token."""
    if longest == 0:
        return [0] * n
    out = [max(1, round(longest * (i + 1) / n) - (7 * i % 13 if i + 1 < n else 0)) for i in range(n)]
    if n >= 8:
        out[0], out[1] = 0, 1
    return out


def _new_lengths(case):
    return [1] * case["n"] if case["new"] == 1 else _lengths(case["n"], case["new"])


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


def _cache(case, g, seed):
    """A pool in use: pages in random order, stale codes where no sequence has written yet."""
    page, n, bits, Hk, D = case["page"], case["n"], case["bits"], case["Hk"], case["D"]
    lengths = _dealt(_lengths(n, case["held"]), seed)
    need = [-(-x // page) for x in lengths]
    new = _new_lengths(case) if case["op"] == "append" else [0]
    pool = sum(need) + 8 + (sum(-(-x // page) + 1 for x in new) if case["op"] == "append" else 0)
    width = max(1, -(-(max(lengths) + max(new)) // page))
    order = torch.randperm(pool, generator=g, device="cuda").int()
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i in range(n):
        table[i, :need[i]] = order[at:at + need[i]]
        at += need[i]
    free = torch.full((pool,), -1, dtype=torch.int32, device="cuda")
    free[:pool - at] = order[at:]
    # codes of normal numbers about the middle and steps about the size that a group of 32 gives, of either sign; what a channel
    # stands out by is in the steps of its group
    half = 1 << (bits - 1)

    def codes():
        out = torch.empty((pool, Hk, page, D * bits // 8), dtype=torch.uint8, device="cuda")
        flat = out.view(-1)
        for i in range(0, flat.numel(), 1 << 27):
            part = flat[i:i + (1 << 27)]
            c = (torch.randn((8 // bits, part.numel()), generator=g, device="cuda") * (half / 2.2)).round_().clamp_(-half, half - 1) + half
            part.copy_(c[0] + (16 * c[1] if bits == 4 else 0))
        return out

    def steps(std):
        size = 2.2 / half * std * torch.exp(0.2 * torch.randn((pool, Hk, page, D // 32), generator=g, device="cuda"))
        return torch.where(torch.rand(size.shape, generator=g, device="cuda") < 0.5, size, -size).half()

    return dict(k_codes=codes(), v_codes=codes(), k_steps=steps(1.0), v_steps=steps(1.0), table=table,
                lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), free_pages=free,
                free_range=torch.tensor([0, pool - at], dtype=torch.int32, device="cuda"),
                shortfall=torch.zeros(1, dtype=torch.int32, device="cuda")), lengths


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, op = _DTYPES[case["dtype"]], case["op"]
    state = dict(op=op, dtype=dt)
    if op == "norm":
        shape = (case["rows"], case["C"])
        state.update(mode=case["mode"], group=case["group"], x=_randn(g, shape, dt), residual=None, weight=None, grads=None)
        if case["residual"]:        # a stream that has grown over the layers, some channels far ahead of the others
            ahead = torch.exp(torch.randn(case["C"], generator=g, device="cuda"))
            state["residual"] = (_randn(g, shape, torch.float32) * ahead).to(dt)
        if case["rows"] >= 8:       # a row of padding
            state["x"][3] = 0
            if case["residual"]:
                state["residual"][3] = 0
        if case["weight"]:
            state["weight"] = (1 + _randn(g, (case["C"],), torch.float32, 0.2)).to(dt)
        if case["mode"] == "train":
            state["grads"] = [_randn(g, shape, dt) for _ in range(2 if case["residual"] else 1)]
        return state
    state["cache"], lengths = _cache(case, g, seed)
    state["bits"] = case["bits"]
    if op == "append":
        new = _dealt(_new_lengths(case), seed + 1)
        shape = (sum(new), case["Hk"], case["D"])
        ahead = torch.exp(0.5 * torch.randn(shape[1:], generator=g, device="cuda"))       # (some channels of the keys stand out)
        state.update(k=(_randn(g, shape, torch.float32) * ahead).to(dt), v=_randn(g, shape, dt), offsets=_offsets(new))
    elif op == "read":
        state.update(offsets=_offsets(lengths), tokens=sum(lengths))
    else:
        state["q"] = _randn(g, (case["n"], case["Hk"] * case["G"], case["D"]), dt)
    return state


# ---- one pass ------------------------------------------------------------------------------------------------------
def _run_own(state):
    from nitrix_b200 import nn

    op = state["op"]
    if op == "norm":
        x, residual, weight = state["x"], state["residual"], state["weight"]
        if state["mode"] == "eight":
            return list(nn.rms_norm_quantized(x, weight, residual=residual, eps=_EPS, group_size=state["group"] or None))
        if state["mode"] == "forward":
            out = nn.rms_norm(x, weight, residual=residual, eps=_EPS)
            return [out] if residual is None else list(out)
        leaves = [t for t in (x, residual, weight) if t is not None]
        for t in leaves:
            t.requires_grad_(True)
        out = nn.rms_norm(x, weight, residual=residual, eps=_EPS)
        out = [out] if residual is None else list(out)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, leaves, state["grads"])]
    cache = nn.QuantizedCache(**state["cache"])
    if op == "decode":
        return [nn.decode_attention(state["q"], cache)]
    if op == "read":
        return list(nn.cache_read(cache, state["offsets"], state["tokens"], dtype=state["dtype"]))
    after = nn.cache_append(cache, state["k"], state["v"], state["offsets"])
    k, v = nn.cache_read(after, state["offsets"], state["k"].shape[0], starts=cache.lengths, dtype=state["dtype"])
    return [k, v, after.table, after.lengths, after.free_range, after.shortfall]


@torch.no_grad()
def run(state):
    if own:
        with torch.enable_grad():
            return _run_own(state)
    return {"norm": _plain_norm, "append": _plain_append, "read": _plain_read, "decode": _plain_decode}[state["op"]](state)


def _plain_norm(state):
    x, residual, weight = state["x"], state["residual"], state["weight"]
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    y = h.float()
    rstd = torch.rsqrt(y.square().mean(-1, keepdim=True) + _EPS)
    unit = y * rstd
    y = unit if weight is None else unit * weight.float()
    stream = [] if residual is None else [h]
    if state["mode"] == "eight":
        groups = y.unflatten(-1, (-1, state["group"] or y.shape[-1]))
        top = groups.abs().amax(-1, keepdim=True).clamp(min=_LEAST)
        codes = (groups * (448 / top)).to(torch.float8_e4m3fn).flatten(-2)
        return [codes, (top / 448).squeeze(-1), *stream]
    out = [y.to(x.dtype), *stream]
    if state["mode"] == "forward":
        return out
    dy = state["grads"][0].float()
    d = dy if weight is None else dy * weight.float()
    dh = rstd * (d - unit * (d * unit).mean(-1, keepdim=True))
    if residual is not None:
        dh = dh + state["grads"][1].float()
        out.append(dh.to(x.dtype))
    out.append(dh.to(x.dtype))
    if weight is not None:
        out.append((dy * unit).sum(0).to(weight.dtype))
    return out


def _unpacked(codes, steps, bits):
    """Values, fp32, of rows of codes and their steps."""
    groups = steps.shape[-1]
    c = codes.unflatten(-1, (8, groups, bits // 2))
    if bits == 4:
        c = torch.stack([c & 15, c >> 4], dim=-1).flatten(-2)
    values = (c.float() - (1 << (bits - 1))) * steps.float()[..., None, :, None]
    return values.transpose(-3, -2).flatten(-3)


def _quantized(x, bits):
    """Rows of codes, and their steps."""
    half = 1 << (bits - 1)
    groups = x.float().unflatten(-1, (-1, 32))
    high, low = groups.amax(-1), groups.amin(-1)
    step = (torch.where(high >= -low, high, low) / -half).clamp(-65504.0, 65504.0).half()
    inverse = torch.where(step == 0, torch.zeros((), device="cuda"), 1 / step.float())
    c = (torch.round(groups * inverse[..., None]) + half).clamp(0, 2 * half - 1).to(torch.uint8)
    c = c.unflatten(-1, (8, 4)).transpose(-3, -2)
    if bits == 4:
        c = c[..., 0::2] | (c[..., 1::2] << 4)
    return c.flatten(-3), step


def _rows_of(cache, offsets, starts, tokens):
    """The page and slot of packed row t, which is token starts[i] + t - offsets[i] of its sequence i."""
    page = cache["k_codes"].shape[2]
    t = torch.arange(tokens, device="cuda")
    row = torch.searchsorted(offsets[1:].contiguous(), t, right=True)
    at = starts[row] + t - offsets[row]
    return cache["table"].long()[row, at // page], at % page


def _plain_append(state):
    c, bits = state["cache"], state["bits"]
    page, width, pool = c["k_codes"].shape[2], c["table"].shape[1], c["k_codes"].shape[0]
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
    c["table"].copy_(torch.where(is_new, fresh, c["table"].long()))
    target, slot = _rows_of(c, offsets, held, state["k"].shape[0])      # (the pools of these cases hold every token)
    out = []
    for name in ("k", "v"):
        codes, steps = _quantized(state[name], bits)
        c[name + "_codes"][target, :, slot] = codes
        c[name + "_steps"][target, :, slot] = steps
        out.append(_unpacked(c[name + "_codes"][target, :, slot], c[name + "_steps"][target, :, slot], bits).to(state["dtype"]))
    free_range = torch.stack([begin + got.sum(), end]).int()
    return [*out, c["table"], lengths.int(), free_range, (want - lengths).sum().int()[None]]


def _plain_read(state):
    c = state["cache"]
    page, slot = _rows_of(c, state["offsets"].long(), torch.zeros_like(c["lengths"]).long(), state["tokens"])
    return [_unpacked(c[name + "_codes"][page, :, slot], c[name + "_steps"][page, :, slot], state["bits"]).to(state["dtype"])
            for name in ("k", "v")]


def _plain_decode(state):
    c, q = state["cache"], state["q"]
    (n, H, D), (_, Hk, page, _) = q.shape, c["k_codes"].shape
    table = torch.clamp(c["table"].long(), min=0)
    most = table.shape[1] * page
    keep = (torch.arange(most, device="cuda") < c["lengths"][:, None])[:, None, None]

    def gathered(name):      # (sequences, heads, tokens, D), behind the last token zeros
        codes = c[name + "_codes"][table].transpose(1, 2).flatten(2, 3)
        steps = c[name + "_steps"][table].transpose(1, 2).flatten(2, 3)
        return _unpacked(codes, torch.where(keep[:, 0, :, :, None], steps, torch.zeros((), dtype=steps.dtype, device="cuda")), state["bits"])

    s = (q.float().view(n, Hk, H // Hk, D) @ gathered("k").transpose(2, 3)) / math.sqrt(D)
    s = torch.where(keep, s, torch.full((), -math.inf, device="cuda"))
    top = s.amax(-1, keepdim=True)
    p = torch.where(keep, torch.exp(s - top), torch.zeros((), device="cuda"))
    total = p.sum(-1, keepdim=True)
    out = (p @ gathered("v")) / torch.where(total > 0, total, torch.ones_like(total))
    return [out.view(n, H, D).to(q.dtype)]


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    esz, op = _BYTES[case["dtype"]], case["op"]
    if op == "norm":
        n = case["rows"] * case["C"]
        streams = 2 if case["residual"] else 1          # x and residual in, y and their sum out
        weight = case["C"] * esz if case["weight"] else 0
        if case["mode"] == "eight":
            scales = 4 * (n // case["group"] if case["group"] else case["rows"])
            return {"bytes": n * (streams * esz + 1 + (streams - 1) * esz) + scales + weight, "flops": 6 * n}
        if case["mode"] == "forward":
            return {"bytes": 2 * streams * n * esz + weight, "flops": 4 * n}
        # and in the backward pass dy, the sum and its gradient in, the gradient (one for both operands) out
        return {"bytes": (2 * streams + streams + 2) * n * esz + 3 * weight, "flops": 14 * n}
    row = 2 * case["Hk"] * (case["D"] * case["bits"] // 8 + case["D"] // 16)        # a token's codes and steps
    dense = 2 * case["Hk"] * case["D"] * esz
    if op == "append":
        tokens = sum(_new_lengths(case))
        return {"bytes": 2 * tokens * (row + dense) + 24 * case["n"], "flops": 0}
    held = _lengths(case["n"], case["held"])
    pages = 4 * sum(-(-x // case["page"]) for x in held)
    if op == "read":
        return {"bytes": sum(held) * (row + dense) + pages, "flops": 0}
    q = case["n"] * case["Hk"] * case["G"] * case["D"]
    return {"bytes": sum(held) * row + 2 * q * esz + pages, "flops": 4 * sum(held) * case["Hk"] * case["G"] * case["D"]}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    with torch.enable_grad():
        return {"norm": _exact_norm, "append": _exact_append, "read": _exact_read, "decode": _exact_decode}[case["op"]](state)


def _exact_norm(state):
    """Gradients by differentiation; the sum of the streams is what is stored of it."""
    train, C = state["mode"] == "train", state["x"].shape[1]
    x = state["x"].double()
    if state["residual"] is not None:
        x = (x + state["residual"].double()).to(state["x"].dtype).double()
    h = x.detach().requires_grad_(train)
    w = torch.ones(C, dtype=torch.float64, device="cuda") if state["weight"] is None else state["weight"].detach().double()
    w.requires_grad_(train)
    y = h * w * torch.pow(torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / C + _EPS, -0.5)
    stream = [] if state["residual"] is None else [h.detach()]
    if state["mode"] == "eight":
        size = state["group"] or C
        parts = y.view(y.shape[0], C // size, size)
        scale = parts.abs().max(dim=2).values.clamp(min=_LEAST) / 448
        # e4m3: three bits behind the leading one, 2^-9 at the least
        z = parts / scale[..., None]
        ulp = torch.exp2(torch.clamp(torch.frexp(z).exponent.double() - 4, min=-9))
        return [(torch.round(z / ulp) * ulp).view_as(y), scale, *stream]
    out = [y.detach(), *stream]
    if train:
        dh, dw = torch.autograd.grad(y, [h, w], state["grads"][0].double())
        if stream:
            dh = dh + state["grads"][1].double()
            out.append(dh)
        out.append(dh)
        if state["weight"] is not None:
            out.append(dw)
    return out


def _exact_values(codes, steps, bits):
    """Element 32 g + 4 j + i of a row, by its place in it."""
    groups = steps.shape[-1]
    d = torch.arange(32 * groups, device="cuda")
    g, j, i = d // 32, d % 32 // 4, d % 4
    byte = (j * groups + g) * (bits // 2) + (i // 2 if bits == 4 else i)
    c = torch.index_select(codes, -1, byte).long()
    if bits == 4:
        c = torch.where(i % 2 == 1, c // 16, c % 16)
    return (c - 2 ** (bits - 1)).double() * torch.index_select(steps, -1, g).double()


def _exact_append(state):
    """What a value becomes: the multiple of its group's step next to it, of those that have a code.  Which of two is the next one
    is part of the definition, in the 32 bits of the quotient."""
    half = 2 ** (state["bits"] - 1)
    out = []
    for name in ("k", "v"):
        x = state[name].double()
        parts = x.view(*x.shape[:-1], x.shape[-1] // 32, 32)
        size = parts.abs().max(dim=-1)
        first = parts.gather(-1, size.indices[..., None])[..., 0]
        top = torch.where(parts.max(dim=-1).values == size.values, size.values, first)
        step = (top / -half).half().double()[..., None]
        quotient = (parts * (1 / step).float().double()).float().double()
        codes = torch.where(step == 0, torch.zeros_like(parts), torch.round(quotient))
        out.append((codes.clamp(-half, half - 1) * step).view_as(x))
    return [*out, None, None, None, None]


def _exact_read(state):
    c = state["cache"]
    page = c["k_codes"].shape[2]
    out = ([], [])
    for i, length in enumerate(c["lengths"].tolist()):
        at = torch.arange(length, device="cuda")
        pages, slots = c["table"][i].long()[at // page], at % page
        for parts, name in zip(out, ("k", "v")):
            parts.append(_exact_values(c[name + "_codes"][pages, :, slots], c[name + "_steps"][pages, :, slots], state["bits"]))
    return [torch.cat(parts) for parts in out]


def _exact_decode(state):
    c, q = state["cache"], state["q"]
    (n, H, D), (_, Hk, page, _) = q.shape, c["k_codes"].shape
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for i, length in enumerate(c["lengths"].tolist()):
        if length == 0:
            continue
        at = torch.arange(length, device="cuda")
        pages, slots = c["table"][i].long()[at // page], at % page
        for h in range(Hk):
            heads = slice(h * (H // Hk), (h + 1) * (H // Hk))
            k, v = (_exact_values(c[name + "_codes"][pages, h, slots], c[name + "_steps"][pages, h, slots], state["bits"]) for name in ("k", "v"))
            out[i, heads] = torch.softmax(torch.einsum("gd,td->gt", q[i, heads].double(), k) * D ** -0.5, dim=-1) @ v
    return [out]
