"""The paged cache in 4 and 8 bits on the GPU: what is written and read back, its bookkeeping, and the attention over it.

Codes, steps and what they read back as are equal to the oracle's: every rounding of the format is part of it.  Attention: 16-bit
operands on the tensor cores round each probability times its step once to fp16 (2^-11), the result once to its type; scores and sums
are fp32, of terms that are added at most 16 deep before a tree (16 roundings, 2^-20 of the scores' sums of magnitudes, doubled for
the exponential and its quotient; exponentials themselves good to 2^-22).
"""
import random

import pytest
import torch

from oracle import decoder_oracle as D
from oracle import few_bits_oracle as O

pytestmark = pytest.mark.gpu

HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _offsets(lengths):
    return _ints([0, *lengths]).cumsum(0).int()


def _cache(pages, page_size, Hk, dim, bits, sequences, width, layout="heads"):
    """An empty cache whose slots hold codes and steps of an earlier use, NaN steps among them."""
    from nitrix_b200.nn import quantized_cache

    c = quantized_cache(pages, page_size, Hk, dim, bits=bits, sequences=sequences, max_length=width * page_size)
    if layout == "tokens":      # tokens before heads, and room behind the rows
        room = lambda t: torch.zeros(pages, page_size, Hk, 2 * t.shape[3], dtype=t.dtype, device="cuda")[..., :t.shape[3]].transpose(1, 2)
        c = c._replace(k_codes=room(c.k_codes), v_codes=room(c.v_codes), k_steps=room(c.k_steps), v_steps=room(c.v_steps))
    for t in c[:2]:
        t.random_(0, 256)
    for t in c[2:4]:
        t.fill_(float("nan"))
    return c


def _same(a, b):
    """Equal, NaN in the same places."""
    return a.dtype == b.dtype and torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


def _at(cache, row, n):
    """Page and slot of the tokens of a row."""
    page = cache.k_codes.shape[2]
    t = torch.arange(n, device="cuda")
    return cache.table[row].long()[t // page], slice(None), t % page


# ---- writing and reading back ----------------------------------------------------------------------------------------------------
def _values(tokens, Hk, dim, dtype, seed=0):
    """Rows of every kind: normal numbers with channels that stand out, zeros, equal ones, one sign, tiny, huge, ties."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(tokens, Hk, dim, generator=g, device="cuda") * torch.exp(torch.randn(dim, generator=g, device="cuda"))
    kinds = [lambda r: r * 0, lambda r: r * 0 + 2.5, lambda r: r.abs(), lambda r: -r.abs(), lambda r: r * 1e-7, lambda r: r * 1e4,
             lambda r: torch.round(r * 4) / 2, lambda r: r * 0 + (torch.arange(dim, device="cuda") % 2 * 2 - 1.0)]
    for i, kind in enumerate(kinds):
        if i < tokens:
            x[i] = kind(x[i])
    return x.to(dtype)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hk,dim", [(1, 32), (2, 64), (3, 96), (8, 128), (1, 160), (5, 256)])
@pytest.mark.parametrize("page_size,layout", [(16, "heads"), (5, "tokens"), (1, "heads")])
def test_tokens_are_written_and_read_back(bits, dtype, Hk, dim, page_size, layout):
    from nitrix_b200.nn import cache_append, cache_read

    lengths = [23, 0, 1, 9]
    cache = _cache(60, page_size, Hk, dim, bits, 4, 40, layout)
    codes_before = cache.k_codes.clone()
    k, v = _values(33, Hk, dim, dtype), _values(33, Hk, dim, dtype, seed=1).flip(0)
    offsets = _offsets(lengths)
    after = cache_append(cache, k, v, offsets)
    assert after.lengths.tolist() == lengths and after.shortfall.tolist() == [0]
    used = torch.zeros(cache.k_codes.shape[:3], dtype=torch.bool, device="cuda")
    for row, n in enumerate(lengths):
        at, first = _at(after, row, n), int(offsets[row])
        for x, codes, steps in ((k, after.k_codes, after.k_steps), (v, after.v_codes, after.v_steps)):
            want, want_steps = O.quantize(x[first:first + n], bits)
            assert _same(steps[at], want_steps)
            assert torch.equal(codes[at], O.packed_codes(want, bits))
        used[at] = True
    # (nothing beside the new tokens' slots is touched)
    assert torch.equal(after.k_codes[~used], codes_before[~used]) and bool(after.k_steps[~used].isnan().all())
    for out in DTYPES:
        got = cache_read(after, offsets, 33, dtype=out)
        for x, y in zip((k, v), got):
            codes, steps = O.quantize(x, bits)
            assert _same(y, O.values(O.packed_codes(codes, bits), steps, bits).to(out))
    assert cache_read(after, offsets, 33)[0].dtype == torch.bfloat16


@pytest.mark.parametrize("bits", [4, 8])
def test_what_is_not_finite_or_beyond_the_steps(bits):
    from nitrix_b200.nn import cache_append, cache_read

    x = torch.randn(6, 1, 64, device="cuda")
    x[0, 0, 5], x[1, 0, 40], x[2, 0, 0] = float("nan"), float("inf"), -float("inf")
    x[3, 0, 1], x[4, 0, 33] = 3e38, -3e38
    x[5] = 1e-12
    cache = _cache(2, 8, 1, 64, bits, 1, 2)
    after = cache_append(cache, x, x.flip(0), _ints([0, 6]))
    got, _ = cache_read(after, _ints([0, 6]), 6, dtype=torch.float32)
    codes, steps = O.quantize(x, bits)
    want = O.values(O.packed_codes(codes, bits), steps, bits).float()
    assert _same(got, want)
    assert bool(got[0, 0, :32].isnan().all()) and not bool(got[0, 0, 32:].isnan().any())
    half = 1 << (bits - 1)
    assert float(got[3, 0, 1]) == 65504.0 * half and float(got[4, 0, 33]) == -65504.0 * half


@pytest.mark.parametrize("bits", [0, 4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_reading_parts_of_sequences(bits, dtype, layout):
    """From a position on, past the end, before the start, rows of no sequence; of both kinds of cache."""
    from nitrix_b200.nn import cache_append, cache_read, paged_cache

    lengths = [40, 0, 7, 100, 1]
    if bits:
        cache = _cache(40, 8, 2, 64, bits, 5, 20, layout)
    else:
        cache = paged_cache(40, 8, 2, 64, sequences=5, max_length=160, dtype=dtype)
        if layout == "tokens":
            cache = cache._replace(k_pages=torch.empty(40, 8, 2, 64, dtype=dtype, device="cuda").transpose(1, 2),
                                   v_pages=torch.empty(40, 8, 2, 72, dtype=dtype, device="cuda")[..., :64].transpose(1, 2))
        cache.k_pages.fill_(float("nan")), cache.v_pages.fill_(float("nan"))
    k, v = (_values(148, 2, 64, dtype, seed=s) for s in (2, 3))
    offsets = _offsets(lengths)
    cache = cache_append(cache, k, v, offsets)
    held = []
    for x in (k, v):
        if bits:
            codes, steps = O.quantize(x, bits)
            x = O.values(O.packed_codes(codes, bits), steps, bits).to(dtype)
        held.append(x)
    starts, wanted, before, behind = [3, 0, -2, 90, 1], [10, 4, 12, 30, 5], 6, 9
    into = _ints([before, *wanted]).cumsum(0).int()
    tokens = int(into[-1]) + behind
    got = cache_read(cache, into, tokens, starts=_ints(starts), dtype=dtype if bits else None)
    for x, y in zip(held, got):
        want = torch.zeros(tokens, 2, 64, dtype=dtype, device="cuda")
        for i, (n, s, w) in enumerate(zip(lengths, starts, wanted)):
            for j in range(w):
                if 0 <= s + j < n:
                    want[int(into[i]) + j] = x[int(offsets[i]) + s + j]
        assert _same(y, want)
    # fewer rows than the offsets name, and none
    part = cache_read(cache, into, 20, starts=_ints(starts), dtype=dtype)
    assert all(_same(a, b[:20]) for a, b in zip(part, got))
    assert cache_read(cache, into, 0)[0].shape == (0, 2, 64)


# ---- bookkeeping -----------------------------------------------------------------------------------------------------------------
class Pair:
    """The cache and its model side by side; a token is one whole number in every element of its rows, which any step gives exactly."""

    def __init__(self, pages, page_size, sequences, width, Hk, dim, bits, layout):
        self.bits, self.model = bits, D.CacheModel(pages, page_size, sequences, width)
        self.cache, self.next, self.dim = _cache(pages, page_size, Hk, dim, bits, sequences, width, layout), 1, dim

    def append(self, counts):
        from nitrix_b200.nn import cache_append

        new = [[(self.next + sum(counts[:i]) + j) % 200 + 1 for j in range(n)] for i, n in enumerate(counts)]
        self.next += sum(counts)
        flat = torch.tensor([t for row in new for t in row], dtype=torch.float32, device="cuda")
        k = (flat[:, None, None].expand(-1, self.cache.k_codes.shape[1], self.dim) + 0).bfloat16()
        self.cache = cache_append(self.cache, k, -k, _offsets(counts))
        self.model.append(new)

    def fork(self, parents):
        from nitrix_b200.nn import cache_fork

        self.cache = cache_fork(self.cache, _ints(parents))
        self.model.fork(parents)

    def free(self, finished):
        from nitrix_b200.nn import cache_free

        self.cache = cache_free(self.cache, torch.tensor(finished, device="cuda"))
        self.model.fork([-1 if f else i for i, f in enumerate(finished)])

    def compact(self):
        from nitrix_b200.nn import cache_compact

        self.cache = cache_compact(self.cache)
        self.model.compact()

    def check(self):
        from nitrix_b200.nn import cache_read

        c, m = self.cache, self.model
        assert c.lengths.tolist() == m.lengths and c.shortfall.tolist() == [m.shortfall]
        begin, end = c.free_range.tolist()
        assert c.free_pages.tolist()[begin:end] == m.free
        for row, (pages, length) in enumerate(zip(c.table.tolist(), m.lengths)):
            used = -(-length // m.page_size)
            assert pages[:used] == m.table[row][:used]
        held = [t for row in range(len(m.lengths)) for t in m.tokens(row)]
        k, v = cache_read(c, _offsets(m.lengths), len(held), dtype=torch.float32)
        want = torch.tensor(held, dtype=torch.float32, device="cuda")[:, None, None].expand_as(k)
        assert torch.equal(k, want) and torch.equal(v, -want)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("page_size,Hk,dim,layout", [(1, 2, 32, "heads"), (3, 1, 96, "tokens"), (16, 8, 128, "heads"), (64, 2, 64, "tokens"), (5, 1, 256, "heads")])
def test_a_random_life(bits, page_size, Hk, dim, layout):
    rng = random.Random(page_size * 1000 + dim + bits)
    pair = Pair(97, page_size, 9, 12, Hk, dim, bits, layout)
    for _ in range(30):
        n = len(pair.model.lengths)
        what = rng.choice(["token", "token", "prompt", "fork", "free", "compact"])
        if what == "token":
            pair.append([rng.choice([0, 1]) for _ in range(n)])
        elif what == "prompt":
            pair.append([rng.choice([0, 0, 1, rng.randint(0, 3 * page_size)]) for _ in range(n)])
        elif what == "fork":
            pair.fork([rng.randint(-1, n - 1) for _ in range(rng.randint(5, 12))])
        elif what == "free":
            pair.free([rng.random() < 0.4 for _ in range(n)])
        else:
            pair.compact()
        pair.check()


def test_pages_and_rows_of_the_table_run_out():
    pair = Pair(5, 4, 3, 4, 2, 64, 4, "heads")
    pair.append([6, 6, 6])
    pair.check()
    assert pair.cache.shortfall.tolist() == [2]
    pair.fork([0, 0, 1])
    pair.check()
    pair = Pair(50, 4, 2, 3, 1, 32, 8, "heads")
    pair.append([20, 5])
    pair.check()
    assert pair.cache.lengths.tolist() == [12, 5]


def test_numbers_that_make_no_sense_stay_in_bounds():
    """Broken tables, lengths, lists, offsets and starts lead to no access outside the pool."""
    from nitrix_b200.nn import cache_append, cache_compact, cache_fork, cache_read, decode_attention

    c = _cache(10, 4, 2, 64, 4, 3, 4)
    k = torch.ones(6, 2, 64, device="cuda")
    good = _ints([0, 2, 4, 6])
    c = cache_append(c, k, k, good)
    bad = [c._replace(table=torch.full_like(c.table, x)) for x in (-7, 10, 1 << 30)]
    bad += [c._replace(lengths=torch.full_like(c.lengths, x)) for x in (-5, 1 << 30, 2 ** 31 - 1)]
    bad += [c._replace(free_range=_ints(x)) for x in ([-9, 400], [8, 2], [10, 10])]
    bad += [c._replace(free_pages=torch.full_like(c.free_pages, x)) for x in (-1, 1 << 29)]
    for cache in bad:
        cache_append(cache, k, k, good)
        cache_fork(cache, _ints([0, 0, 5, 1]))
        cache_compact(cache)
        cache_read(cache, good, 6)
        decode_attention(torch.ones(3, 2, 64, device="cuda").half(), cache)
        decode_attention(torch.ones(3, 2, 64, device="cuda"), cache)
    for offsets in ([0, 9, 2, 6], [-4, 1, 2, 3], [5, 6, 6, 100], [0, 0, 0, 0], [2 ** 31 - 1] * 4, [-2 ** 31] * 4):
        cache_append(c, k, k, _ints(offsets))
        for starts in (None, _ints([2 ** 31 - 1, -2 ** 31, 5])):
            cache_read(c, _ints(offsets), 6, starts=starts)
    torch.cuda.synchronize()


# ---- attention of one token ---------------------------------------------------------------------------------------------------------
def _filled(lengths, page_size, Hk, dim, bits, seed=0, layout="heads", std=1.0):
    """A cache of random codes and steps of either sign in pages of random order; NaN steps wherever no token is."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page_size) for n in lengths]
    c = _cache(sum(need) + 3, page_size, Hk, dim, bits, len(lengths), max(1, max(need, default=1)), layout)
    order = torch.randperm(sum(need) + 3, generator=g, device="cuda").int()
    at = 0
    for i, n in enumerate(lengths):
        c.table[i, :need[i]] = order[at:at + need[i]]
        at += need[i]
        where = _at(c, i, n)
        for codes, steps in ((c.k_codes, c.k_steps), (c.v_codes, c.v_steps)):
            x = torch.randn(n, Hk, dim, generator=g, device="cuda") * std
            a, b = O.quantize(x, bits)
            codes[where], steps[where] = O.packed_codes(a, bits), b
    c.lengths.copy_(_ints(lengths))
    return c


def _check_decode(q, cache, lengths, bits, scale=None, spoiled=None):
    """``spoiled``: the elements that have to be NaN; all others must be good."""
    from nitrix_b200.nn import decode_attention

    got = decode_attention(q, cache, scale=scale)
    k, v = O.cache_values(cache, bits)
    want, spread, reach = O.decode(q, k, v, cache.table, lengths, q.shape[-1] ** -0.5 if scale is None else scale)
    assert got.dtype == q.dtype and got.shape == q.shape
    assert torch.equal(got.isnan(), torch.zeros_like(got, dtype=torch.bool) if spoiled is None else spoiled)
    p_rounding = 0 if q.dtype == torch.float32 else 2.0 ** -11
    bound = HALF[q.dtype] * want.abs() + (p_rounding + 2 * 16 * 2.0 ** -24 * (1 + reach) + 2.0 ** -20) * 2 * spread
    err = ((got.double() - want).abs() - bound - 2.0 ** -25)[~got.isnan()]
    assert float(err.max()) <= 0, float(err.max())
    return got


LENGTHS = {"mixed": [0, 1, 15, 16, 17, 63, 64, 65, 129, 300], "one": [1], "empty": [0, 0, 0], "long": [5000], "two": [2000, 7]}


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 32, 96, 256])
@pytest.mark.parametrize("Hk,G", [(1, 1), (2, 3), (4, 8), (1, 9), (2, 16), (1, 33)])
@pytest.mark.parametrize("name,page_size", [("mixed", 16), ("mixed", 5), ("one", 1), ("empty", 32), ("long", 128), ("two", 64)])
def test_decode(bits, dtype, dim, Hk, G, name, page_size):
    lengths = LENGTHS[name]
    cache = _filled(lengths, page_size, Hk, dim, bits, seed=dim + G)
    q = torch.randn(len(lengths), Hk * G, dim, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    got = _check_decode(q, cache, lengths, bits)
    for i, n in enumerate(lengths):
        if n == 0:
            assert not bool(got[i].any())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_peaked_scores_and_scales(bits, dtype):
    """Scores far apart (one key takes all), equal ones, a negative scale; queries of any size, zeros among them."""
    lengths = [700, 33, 5]
    cache = _filled(lengths, 16, 2, 64, bits)
    q = torch.randn(3, 8, 64, device="cuda").to(dtype)
    for scale in (4.0, 0.0, -0.125, 1e-35):
        _check_decode(q, cache, lengths, bits, scale)
    for size in (6e-8, 1e-3, 6e3, 0.0):
        _check_decode((q.float() * size).to(dtype), cache, lengths, bits, 1 / 64 if size < 1 else 0.25 / size)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_values_of_very_different_size(bits, dtype, dim):
    """The attended tokens' values are small beside those of tokens that get no weight; groups of a row differ as much."""
    lengths = [300, 40]
    cache = _filled(lengths, 16, 2, dim, bits)
    g = torch.Generator(device="cuda").manual_seed(9)
    size = torch.exp2(torch.randint(-9, 9, cache.v_steps.shape, generator=g, device="cuda").float())
    cache.v_steps.copy_((cache.v_steps.float() * size).half())
    _check_decode(torch.randn(2, 4, dim, device="cuda").to(dtype), cache, lengths, bits, 0.02)
    # one token takes all the weight; its values are the smallest
    cache = _filled(lengths, 16, 2, dim, bits)
    where = _at(cache, 0, 300)
    cache.v_steps[where] = cache.v_steps[where] * 100
    first = tuple(x if isinstance(x, slice) else x[:1] for x in where)
    cache.v_steps[first] = cache.v_steps[first] * 1e-4
    k, _ = O.cache_values(cache, bits)
    q = k[where[0][0], :, where[2][0]][None].repeat_interleave(2, 1).expand(2, 4, dim).to(dtype)
    got = _check_decode(q, cache, lengths, bits, 3.0)
    assert float(got[0].float().abs().max()) < 0.1


def test_decode_what_is_not_finite_stays_in_its_group():
    """A step that is NaN spoils what it stands in, nothing else.  (What the others are rounded at goes by the largest step of a token's
    values, so that they need not be the same bits as without it.)"""
    lengths = [50, 20]
    for bits in (4, 8):
        for dtype in DTYPES:
            cache = _filled(lengths, 16, 2, 64, bits)
            q = torch.randn(2, 4, 64, device="cuda").to(dtype)
            spoiled = torch.zeros(2, 4, 64, dtype=torch.bool, device="cuda")
            page, slot = int(cache.table[0, 1]), 3      # token 19 of the first sequence, of key head 1 the second group
            cache.v_steps[page, 1, slot, 1] = float("nan")
            spoiled[0, 2:, 32:] = True
            _check_decode(q, cache, lengths, bits, spoiled=spoiled)
            cache.k_steps[page, 0, slot, 0] = float("nan")
            spoiled[0, :2] = True
            _check_decode(q, cache, lengths, bits, spoiled=spoiled)


def test_decode_layouts_and_misaligned_queries():
    lengths = [100, 31, 64]
    for layout in ("heads", "tokens"):
        cache = _filled(lengths, 16, 2, 64, 4, layout=layout)
        wide = torch.randn(3, 24, 64, device="cuda").bfloat16()
        _check_decode(wide[:, 4:12], cache, lengths, 4)
        _check_decode(wide.view(-1)[1:1 + 3 * 8 * 64].view(3, 8, 64), cache, lengths, 4)
        _check_decode(wide[:, :1].expand(3, 8, 64), cache, lengths, 4)


@pytest.mark.parametrize("bits", [4, 8])
def test_decode_many_sequences_and_an_uneven_split(bits):
    rng = random.Random(0)
    lengths = [rng.choice([0, 1, rng.randint(1, 400)]) for _ in range(321)] + [9000]
    cache = _filled(lengths, 16, 1, 64, bits)
    _check_decode(torch.randn(322, 4, 64, device="cuda").half(), cache, lengths, bits)


@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_beyond_32_bits(dtype):
    """A pool of more than 2^32 bytes of codes; the pages in use lie at its end."""
    from nitrix_b200.nn import cache_append, cache_compact, cache_fork, cache_read, decode_attention

    page, Hk, dim = 64, 8, 128
    pool = (1 << 32) // (page * Hk * dim // 2) + 100
    cache = _cache(2, page, Hk, dim, 4, 2, 8)
    codes = torch.empty(pool, Hk, page, dim // 2, dtype=torch.uint8, device="cuda")
    steps = torch.empty(pool, Hk, page, dim // 32, dtype=torch.float16, device="cuda")
    cache = cache._replace(k_codes=codes, v_codes=torch.empty_like(codes), k_steps=steps, v_steps=torch.empty_like(steps),
                           free_pages=torch.arange(pool - 1, -1, -1, dtype=torch.int32, device="cuda"), free_range=_ints([0, pool]))
    k, v = (torch.randn(470, Hk, dim, device="cuda").to(dtype) for _ in range(2))
    cache = cache_append(cache, k, v, _ints([0, 270, 470]))
    assert cache.table[0, :5].tolist() == list(range(pool - 1, pool - 6, -1))
    q = torch.randn(3, Hk, dim, device="cuda").to(dtype)
    whole, want = cache_read(cache, _ints([0, 270, 470]), 470, dtype=dtype), decode_attention(q[:2], cache)
    small = cache._replace(**{n: getattr(cache, n)[-16:].clone() for n in ("k_codes", "v_codes", "k_steps", "v_steps")}, table=cache.table - (pool - 16))
    assert torch.equal(decode_attention(q[:2], small), want)
    assert all(torch.equal(a, b) for a, b in zip(cache_read(small, _ints([0, 270, 470]), 470, dtype=dtype), whole))
    packed = cache_compact(cache_fork(cache, _ints([1, 1, 0])))
    assert int(packed.table.max()) < 16
    got = cache_read(packed, _ints([0, 200, 400, 670]), 670, dtype=dtype)
    for a, b in zip(got, whole):
        assert torch.equal(a, torch.cat([b[270:], b[270:], b[:270]]))


def test_the_same_every_time():
    from nitrix_b200.nn import decode_attention

    lengths = [3000, 1, 777]
    cache = _filled(lengths, 16, 4, 128, 4)
    for dtype in DTYPES:
        q = torch.randn(3, 16, 128, device="cuda").to(dtype)
        first = decode_attention(q, cache)
        for _ in range(5):
            assert torch.equal(decode_attention(q, cache), first)


@pytest.mark.parametrize("bits", [4, 8])
def test_a_generation_step_in_a_graph(bits):
    """Append, reading back and attention captured once, replayed with other tokens; lengths move on the device."""
    from nitrix_b200.nn import cache_append, cache_read, decode_attention

    cache = _cache(64, 4, 2, 64, bits, 3, 10)
    k, v = (torch.randn(3, 2, 64, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(3, 4, 64, device="cuda").bfloat16()
    offsets = torch.arange(4, device="cuda").int()

    def step():
        after = cache_append(cache, k, v, offsets)
        new = cache_read(after, offsets, 3, starts=cache.lengths)
        out = decode_attention(q, after)
        cache.lengths.copy_(after.lengths)
        cache.free_range.copy_(after.free_range)
        return out, new
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, new = step()
    for n in range(2, 12):
        for t in (k, v, q):
            t.copy_(torch.randn_like(t))
        graph.replay()
        torch.cuda.synchronize()
        assert cache.lengths.tolist() == [n] * 3
        codes, steps = O.quantize(k, bits)
        assert torch.equal(new[0], O.values(O.packed_codes(codes, bits), steps, bits).bfloat16())
        assert torch.equal(out, decode_attention(q, cache))
        _check_decode(q, cache, [n] * 3, bits)


def test_an_earlier_cache_stays_valid_and_versions_rise():
    from nitrix_b200.nn import cache_append, cache_compact, cache_fork, cache_free, cache_read

    pair = Pair(40, 4, 4, 8, 2, 64, 4, "heads")
    pair.append([9, 3, 0, 6])
    before = pair.cache
    k = torch.full((8, 2, 64), 177.0, device="cuda")

    def rises(call):
        old = [t._version for t in before[:4]]
        call()
        return [t._version > o for t, o in zip(before[:4], old)]
    assert all(rises(lambda: cache_append(before, k, k, _ints([0, 2, 4, 6, 8]))))
    pair.check()
    assert all(rises(lambda: cache_fork(before, _ints([0, 0, 1, 1, 3, 3]))))
    pair.check()
    assert all(rises(lambda: cache_compact(before)))
    pair.check()
    assert not any(rises(lambda: cache_free(before, torch.zeros(4, dtype=torch.bool, device="cuda"))))
    assert not any(rises(lambda: cache_read(before, _ints([0, 1, 2, 3, 4]), 4)))


def test_refusals():
    from nitrix_b200.nn import QuantizedCache, cache_append, cache_compact, cache_fork, cache_read, decode_attention, paged_cache, quantized_cache

    cache = quantized_cache(8, 4, 2, 64, sequences=3, max_length=16)
    k = torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    offsets = torch.arange(4, device="cuda").int()
    q = torch.zeros(3, 4, 64, device="cuda", dtype=torch.bfloat16)
    calls = [lambda c: cache_append(c, k, k, offsets), lambda c: cache_fork(c, offsets[:3]), cache_compact, lambda c: cache_read(c, offsets, 3),
             lambda c: decode_attention(q, c)]
    for call in calls:
        with pytest.raises(TypeError, match="CUDA tensor"):
            call(QuantizedCache(*(t.cpu() for t in cache)))
        with pytest.raises(TypeError, match="uint8"):
            call(cache._replace(k_codes=cache.k_codes.char()))
        with pytest.raises(TypeError, match="v_codes"):
            call(cache._replace(v_codes=cache.v_codes.char()))
        with pytest.raises(ValueError, match="one shape"):
            call(cache._replace(v_codes=cache.v_codes[:4]))
        with pytest.raises(TypeError, match="float16"):
            call(cache._replace(k_steps=cache.k_steps.float()))
        with pytest.raises(ValueError, match="steps"):
            call(cache._replace(v_steps=cache.v_steps[:, :1]))
        with pytest.raises(ValueError, match="bits"):
            call(cache._replace(k_steps=cache.k_steps.repeat(1, 1, 1, 3), v_steps=cache.v_steps.repeat(1, 1, 1, 3)))
        with pytest.raises(ValueError, match="unit stride"):
            call(cache._replace(k_codes=cache.k_codes.transpose(2, 3).contiguous().transpose(2, 3)))
        with pytest.raises(ValueError, match="unit stride"):
            call(cache._replace(k_steps=cache.k_steps.transpose(2, 3).contiguous().transpose(2, 3)))
        with pytest.raises(ValueError, match="expanded"):
            call(cache._replace(k_steps=cache.k_steps[:1].expand(8, 2, 4, 2)))
        with pytest.raises(RuntimeError, match="16-byte"):
            call(cache._replace(k_codes=torch.zeros(8 * 2 * 4 * 32 + 1, dtype=torch.uint8, device="cuda")[1:].view(8, 2, 4, 32)))
        with pytest.raises(RuntimeError, match="16-byte"):
            call(cache._replace(v_steps=torch.zeros(8 * 2 * 4 * 2 + 1, dtype=torch.float16, device="cuda")[1:].view(8, 2, 4, 2)))
        with pytest.raises(TypeError, match="table"):
            call(cache._replace(table=cache.table.long()))
        with pytest.raises(ValueError, match="lengths"):
            call(cache._replace(lengths=cache.lengths[:2]))
    with pytest.raises(TypeError, match="k must be"):
        cache_append(cache, k.double(), k.double(), offsets)
    with pytest.raises(TypeError, match="k and v"):
        cache_append(cache, k, k.float(), offsets)
    with pytest.raises(ValueError, match="k and v"):
        cache_append(cache, k[..., :32], k[..., :32], offsets)
    with pytest.raises(TypeError, match="q must be"):
        decode_attention(q.double(), cache)
    with pytest.raises(ValueError, match="q must be"):
        decode_attention(q[:, :3], cache)
    with pytest.raises(NotImplementedError, match="differentiable"):
        decode_attention(q.clone().requires_grad_(True), cache)
    with pytest.raises(RuntimeError, match="256"):
        decode_attention(torch.zeros(1, 1, 288, device="cuda"), quantized_cache(2, 4, 1, 288, sequences=1, max_length=4))
    with pytest.raises(ValueError, match="offsets"):
        cache_read(cache, offsets[:3], 3)
    with pytest.raises(TypeError, match="offsets"):
        cache_read(cache, offsets.long(), 3)
    with pytest.raises(ValueError, match="starts"):
        cache_read(cache, offsets, 3, starts=offsets)
    with pytest.raises(ValueError, match="tokens"):
        cache_read(cache, offsets, -1)
    with pytest.raises(TypeError, match="dtype"):
        cache_read(cache, offsets, 3, dtype=torch.float64)
    with pytest.raises(TypeError, match="dtype"):
        cache_read(paged_cache(8, 4, 2, 64, sequences=3, max_length=16), offsets, 3, dtype=torch.float32)
    dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
    for call in (lambda: decode_attention(dual(q), cache), lambda: cache_append(cache, dual(k), k, offsets), lambda: cache_read(cache._replace(k_steps=dual(cache.k_steps)), offsets, 3)):
        with pytest.raises(NotImplementedError, match="forward-mode"), torch.autograd.forward_ad.dual_level():
            call()


@pytest.mark.parametrize("bits", [4, 8])
def test_every_step(bits):
    """Codes under every fp16 step that there is, of values at, beside and far from the borders between two codes."""
    from nitrix_b200.nn import cache_append

    half = 1 << (bits - 1)
    steps = torch.arange(1, 0x7c00, device="cuda").short().view(torch.float16).float()
    steps = torch.cat([steps, -steps])
    g = torch.Generator(device="cuda").manual_seed(0)
    ratio = torch.randint(-half, half, (steps.numel(), 32), generator=g, device="cuda").float() + 0.5
    ratio[:, 16:] += torch.randn(steps.numel(), 16, generator=g, device="cuda") * 2.0 ** -20
    x = (ratio * steps[:, None]).clamp(-half * steps.abs()[:, None], half * steps.abs()[:, None])
    x[:, 0] = -half * steps      # (the largest, which makes the step)
    x = x[:, None].contiguous()
    cache = _cache(len(steps) // 64 + 2, 64, 1, 32, bits, 1, len(steps) // 64 + 2)
    after = cache_append(cache, x, x, _ints([0, len(steps)]))
    at = _at(after, 0, len(steps))
    want, want_steps = O.quantize(x, bits)
    assert torch.equal(after.k_steps[at], want_steps) and torch.equal(after.k_codes[at], O.packed_codes(want, bits))


def test_lengths_at_the_end_of_32_bits():
    """A table of one page many times over: 2^31 tokens and more.  A sequence counts 2^31 - 256 of them at most."""
    from nitrix_b200.nn import QuantizedCache, cache_append, cache_read, decode_attention

    page, most = 1 << 16, 2 ** 31 - 256
    table, z = torch.zeros(1, (1 << 15) + 4, dtype=torch.int32, device="cuda"), _ints([0])
    for dtype, dim, bits in ((torch.bfloat16, 64, 4), (torch.float16, 128, 8), (torch.float32, 32, 8)):
        codes = torch.full((1, 1, page, dim * bits // 8), 0x99 if bits == 4 else 0x81, dtype=torch.uint8, device="cuda")
        steps = torch.zeros(1, 1, page, dim // 32, dtype=torch.float16, device="cuda")
        for n in (2 ** 31 - 1, most, most - 63):
            cache = QuantizedCache(codes, codes, steps, torch.full_like(steps, 3.0), table, _ints([n]), z, _ints([0, 0]), z)
            out = decode_attention(torch.ones(1, 1, dim, dtype=dtype, device="cuda"), cache)
            assert bool(((out - 3).abs() < 0.02).all()), (dtype, n)
        got, _ = cache_read(cache._replace(k_steps=cache.v_steps, lengths=_ints([most])), _ints([0, 9]), 9, starts=_ints([most - 5]))
        assert bool((got[:5] == 3).all()) and not bool(got[5:].any())
    more = torch.zeros(4, 1, 32, dtype=torch.bfloat16, device="cuda")
    after = cache_append(cache._replace(lengths=_ints([most - 3])), more, more, _ints([0, 4]))
    assert after.lengths.tolist() == [most] and after.shortfall.tolist() == [1]


def test_two_graphs_and_an_eager_call_with_one_cache():
    """Workspaces belong to their calls: graphs replayed in any order, with eager calls between, give what each gave alone."""
    from nitrix_b200.nn import decode_attention

    lengths = [900, 40, 333]
    cache = _filled(lengths, 16, 2, 128, 4)
    q = [torch.randn(3, 8, 128, device="cuda").half() for _ in range(3)]
    want = [decode_attention(x, cache) for x in q]
    graphs = []
    for x in q[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = decode_attention(x, cache)
        graphs.append((graph, out))
    for order in ((0, 1), (1, 0, 1), (0, 0)):
        for i in order:
            graphs[i][0].replay()
            assert torch.equal(decode_attention(q[2], cache), want[2])
        for i in set(order):
            assert torch.equal(graphs[i][1], want[i])


def test_forks_and_compactions_in_a_graph():
    from nitrix_b200.nn import cache_compact, cache_fork

    pair = Pair(64, 4, 6, 8, 2, 64, 4, "heads")
    pair.append([9, 3, 0, 17, 30, 5])
    held = type(pair.cache)(*pair.cache[:4], *(t.clone() for t in pair.cache[4:]))
    parents = torch.arange(6, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache_compact(cache_fork(held, parents))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = cache_compact(cache_fork(held, parents))
    rng = random.Random(5)
    for _ in range(10):
        for mine, theirs in zip(held[4:], pair.cache[4:]):
            mine.copy_(theirs)
        chosen = [rng.randint(-1, 5) for _ in range(6)]
        parents.copy_(_ints(chosen))
        graph.replay()
        pair.cache = type(result)(*held[:4], *(t.clone() for t in result[4:]))
        pair.model.fork(chosen)
        pair.model.compact()
        pair.check()
        pair.append([rng.choice([0, 1, 3]) for _ in range(6)])
        pair.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_large_groups(dtype, dim):
    lengths = [100, 3, 700]
    cache = _filled(lengths, 16, 1, dim, 4)
    _check_decode(torch.randn(3, 130, dim, device="cuda").to(dtype), cache, lengths, 4)


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_a_query_that_is_not_finite_spoils_its_head(dtype):
    lengths = [50, 20]
    for bits in (4, 8):
        cache = _filled(lengths, 16, 2, 64, bits)
        q = torch.randn(2, 12, 64, device="cuda").to(dtype)
        q[0, 3, 5], q[1, 11, 63] = float("nan"), float("nan")
        spoiled = torch.zeros(2, 12, 64, dtype=torch.bool, device="cuda")
        spoiled[0, 3] = spoiled[1, 11] = True
        _check_decode(q, cache, lengths, bits, spoiled=spoiled)


def test_decode_on_another_stream():
    from nitrix_b200.nn import decode_attention

    cache = _filled([900, 40, 0], 16, 2, 64, 4)
    q = torch.randn(3, 8, 64, device="cuda").half()
    want = decode_attention(q, cache)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [decode_attention(q, cache) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, want) for x in got)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_appending_views(bits, dtype):
    """Slices of one projection's output, misaligned rows, one head's row for all heads."""
    from nitrix_b200.nn import cache_append, cache_read

    offsets, n = _ints([0, 5, 19]), 19
    g = torch.Generator(device="cuda").manual_seed(0)
    wide = torch.randn(n, (6 + 2 * 3) * 64, generator=g, device="cuda").to(dtype)
    odd = torch.randn(n * 3 * 64 + 1, generator=g, device="cuda").to(dtype)[1:].view(n, 3, 64)
    heads = wide.unflatten(1, (12, 64))
    for k, v in ((heads[:, 6:9], heads[:, 9:]), (odd, odd.flip(0)), (heads[:, :1].expand(n, 3, 64), odd), (odd.transpose(0, 1).contiguous().transpose(0, 1), heads[:, ::4])):
        cache = _cache(12, 4, 3, 64, bits, 2, 8)
        got = cache_read(cache_append(cache, k, v, offsets), offsets, n, dtype=torch.float32)
        for x, y in zip((k, v), got):
            codes, steps = O.quantize(x, bits)
            assert torch.equal(y, O.values(O.packed_codes(codes, bits), steps, bits).float())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_steps_in_pages_that_lie_far_apart(dtype):
    """Strides from one page's steps to the next's of 2^31 elements."""
    from nitrix_b200.nn import cache_append, cache_read, decode_attention

    small = _cache(2, 16, 2, 128, 4, 1, 2)
    buffer = torch.empty((1 << 31) + 1024, dtype=torch.float16, device="cuda")
    far = lambda at: buffer[at:].as_strided((2, 2, 16, 4), (1 << 31, 64, 4, 1))
    large = small._replace(k_codes=small.k_codes.clone(), v_codes=small.v_codes.clone(), k_steps=far(0), v_steps=far(512), table=small.table.clone())
    k, v = (torch.randn(30, 2, 128, device="cuda").to(dtype) for _ in range(2))
    q, offsets = torch.randn(1, 4, 128, device="cuda").to(dtype), _ints([0, 30])
    small, large = (cache_append(c, k, v, offsets) for c in (small, large))
    assert torch.equal(small.table, large.table)
    assert all(torch.equal(a, b) for a, b in zip(cache_read(small, offsets, 30), cache_read(large, offsets, 30)))
    _check_decode(q, small, [30], 4)
    _check_decode(q, large, [30], 4)
