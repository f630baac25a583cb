"""The paged cache on the GPU against a model in plain Python, and the attention of one token over it against 64 bits.

Whole numbers and moved values are equal.  Attention: probabilities and the result of 16-bit operands are each rounded once to
the operand type, everything else is fp32, so the error is within u (sum p |v| + |out|) with u one ulp's half, doubled for the
fp32 parts: exponentials of scores that are good to 2^-22 relative, sums of up to a few thousand terms.
"""
import random

import pytest
import torch

from oracle import decoder_oracle as O

pytestmark = pytest.mark.gpu

U = {t: torch.finfo(t).eps for t in (torch.bfloat16, torch.float16)} | {torch.float32: 1e-5}


# ---- bookkeeping -----------------------------------------------------------------------------------------------------------
class Pair:
    """The cache and its model side by side; a token is one number, held in every element of its rows."""

    def __init__(self, pages, page_size, sequences, width, Hk=2, D=8, dtype=torch.float32, strided=False):
        from nitrix_b200.nn import paged_cache

        self.model = O.CacheModel(pages, page_size, sequences, width)
        self.cache = paged_cache(pages, page_size, Hk, D, sequences=sequences, max_length=width * page_size, dtype=dtype)
        if strided:      # tokens before heads, and room between the rows
            def pool():
                return torch.zeros(pages, page_size, Hk, 2 * D, dtype=dtype, device="cuda")[..., :D].transpose(1, 2)
            self.cache = self.cache._replace(k_pages=pool(), v_pages=pool())
        self.cache.k_pages.fill_(float("nan"))
        self.cache.v_pages.fill_(float("nan"))
        self.next = 1

    def append(self, counts):
        from nitrix_b200.nn import cache_append

        new = [list(range(self.next + sum(counts[:i]), self.next + sum(counts[:i + 1]))) for i in range(len(counts))]
        self.next = (self.next + sum(counts)) % 199 + 1 if self.cache.k_pages.dtype != torch.float32 else self.next + sum(counts)
        Hk, D = self.cache.k_pages.shape[1], self.cache.k_pages.shape[3]
        flat = torch.tensor([t for row in new for t in row], dtype=torch.float32, device="cuda").to(self.cache.k_pages.dtype)
        k = flat[:, None, None].expand(-1, Hk, D) + 0
        offsets = torch.tensor([0, *counts], device="cuda").cumsum(0).int()
        self.cache = cache_append(self.cache, k, -k, offsets)
        self.model.append(new)

    def fork(self, parents):
        from nitrix_b200.nn import cache_fork

        self.cache = cache_fork(self.cache, torch.tensor(parents, dtype=torch.int32, device="cuda"))
        self.model.fork(parents)

    def free(self, finished):
        from nitrix_b200.nn import cache_free

        self.cache = cache_free(self.cache, torch.tensor(finished, device="cuda"))
        self.model.fork([-1 if f else i for i, f in enumerate(finished)])

    def compact(self):
        from nitrix_b200.nn import cache_compact

        self.cache = cache_compact(self.cache)
        self.model.compact()

    def check(self, listed=True):
        c, m = self.cache, self.model
        assert c.lengths.tolist() == m.lengths
        begin, end = c.free_range.tolist()
        assert c.free_pages.tolist()[begin:end] == m.free
        assert c.shortfall.tolist() == [m.shortfall]
        table, page = c.table.tolist(), m.page_size
        for row, length in enumerate(m.lengths):
            used = -(-length // page)
            assert table[row][:used] == m.table[row][:used]
            if listed:
                assert all(x == -1 for x in table[row][used:])
            at = torch.arange(length, device="cuda")
            pages = c.table[row].long()[at // page]
            want = torch.tensor(m.tokens(row), dtype=torch.float32, device="cuda")[:, None, None].to(c.k_pages.dtype)
            for pool, sign in ((c.k_pages, 1), (c.v_pages, -1)):
                got = pool[pages, :, at % page]
                assert torch.equal(got, (sign * want).expand_as(got)), row


@pytest.mark.parametrize("page_size", [1, 3, 16, 64])
@pytest.mark.parametrize("Hk,D,dtype", [(2, 8, torch.float32), (1, 64, torch.float16), (3, 40, torch.bfloat16), (8, 128, torch.float16)])
@pytest.mark.parametrize("strided", [False, True])
def test_a_random_life(page_size, Hk, D, dtype, strided):
    rng = random.Random(page_size * 1000 + D)
    pair = Pair(97, page_size, 9, 12, Hk, D, dtype, strided)
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


def test_pages_run_out():
    pair = Pair(5, 4, 3, 4)
    pair.append([6, 6, 6])           # two pages each, the last row gets one
    pair.check()
    assert pair.cache.shortfall.tolist() == [2] and pair.cache.lengths.tolist() == [6, 6, 4]
    pair.append([1, 3, 1])           # the second row's third token and the last row's find no page
    pair.check()
    pair.fork([0, 0, 1])             # nothing is free: the second child keeps whole pages
    pair.check()
    assert pair.cache.shortfall.tolist() == [3] and pair.cache.lengths.tolist() == [7, 4, 8]


def test_rows_of_the_table_run_out():
    pair = Pair(50, 4, 2, 3)
    pair.append([20, 5])
    pair.check()
    assert pair.cache.lengths.tolist() == [12, 5] and pair.cache.shortfall.tolist() == [8]
    pair.append([1, 9])
    pair.check()
    pair.compact()
    pair.check()


@pytest.mark.parametrize("sequences", [1, 31, 33, 300, 1500])
def test_many_sequences(sequences):
    rng = random.Random(sequences)
    pair = Pair(4 * sequences + 3, 4, sequences, 6)
    pair.append([rng.randint(0, 9) for _ in range(sequences)])
    pair.check()
    pair.fork([rng.randint(-1, sequences - 1) for _ in range(sequences)])
    pair.check()
    pair.append([1] * sequences)
    pair.check()
    pair.compact()
    pair.check()


def test_an_earlier_cache_stays_valid():
    from nitrix_b200.nn import cache_append, cache_compact, cache_fork

    pair = Pair(40, 4, 4, 8)
    pair.append([9, 3, 0, 6])
    before = pair.cache
    k = torch.full((8, 2, 8), 777.0, device="cuda")
    cache_append(before, k, k, torch.arange(0, 9, 2, device="cuda").int())
    pair.check(listed=False)
    cache_fork(before, torch.tensor([0, 0, 1, 1, 3, 3], dtype=torch.int32, device="cuda"))
    pair.check(listed=False)
    cache_compact(before)
    pair.check(listed=False)


def test_numbers_that_make_no_sense_stay_in_bounds():
    """Broken tables, lengths, lists and offsets lead to no access outside the pool."""
    from nitrix_b200.nn import cache_append, cache_compact, cache_fork, decode_attention

    pair = Pair(10, 4, 3, 4)
    pair.append([5, 6, 7])
    c = pair.cache
    bad = [c._replace(table=torch.full_like(c.table, x)) for x in (-7, 10, 1 << 30)]
    bad += [c._replace(lengths=torch.full_like(c.lengths, x)) for x in (-5, 1 << 30, 2 ** 31 - 1)]
    bad += [c._replace(free_range=torch.tensor(x, dtype=torch.int32, device="cuda")) for x in ([-9, 400], [8, 2], [10, 10])]
    bad += [c._replace(free_pages=torch.full_like(c.free_pages, x)) for x in (-1, 1 << 29)]
    k = torch.ones(6, 2, 8, device="cuda")
    good = torch.tensor([0, 2, 4, 6], dtype=torch.int32, device="cuda")
    for cache in bad:
        cache_append(cache, k, k, good)
        cache_fork(cache, torch.tensor([0, 0, 5, 1], dtype=torch.int32, device="cuda"))
        cache_compact(cache)
        decode_attention(torch.ones(3, 2, 8, device="cuda"), cache)
    for offsets in ([0, 9, 2, 6], [-4, 1, 2, 3], [5, 6, 6, 100], [0, 0, 0, 0]):
        cache_append(c, k, k, torch.tensor(offsets, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()


# ---- attention of one token ---------------------------------------------------------------------------------------------------
def _cache_of(lengths, page_size, Hk, D, dtype, seed=0, stale=float("nan"), spare=3, layout="heads"):
    from nitrix_b200.nn import PagedCache

    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page_size) for n in lengths]
    pool = sum(need) + spare
    width = max(1, max(need, default=1))
    order = torch.randperm(pool, generator=g, device="cuda").int()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")

    def pages():
        if layout == "tokens":
            return torch.full((pool, page_size, Hk, D), stale, dtype=dtype, device="cuda").transpose(1, 2)
        return torch.full((pool, Hk, page_size, D), stale, dtype=dtype, device="cuda")
    k, v = pages(), pages()
    at = 0
    for i, n in enumerate(lengths):
        table[i, :need[i]] = order[at:at + need[i]]
        at += need[i]
        t = torch.arange(n, device="cuda")
        where = table[i].long()[t // page_size], slice(None), t % page_size
        k[where] = torch.randn(n, Hk, D, generator=g, device="cuda").to(dtype)
        v[where] = torch.randn(n, Hk, D, generator=g, device="cuda").to(dtype)
    z = torch.zeros(1, dtype=torch.int32, device="cuda")
    return PagedCache(k, v, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), order, torch.tensor([at, pool], dtype=torch.int32, device="cuda"), z)


def _check_decode(q, cache, lengths, scale=None):
    from nitrix_b200.nn import decode_attention

    got = decode_attention(q, cache, scale=scale)
    want, bound = O.decode(q, cache.k_pages, cache.v_pages, cache.table, lengths, q.shape[-1] ** -0.5 if scale is None else scale)
    assert got.dtype == q.dtype and got.shape == q.shape
    err = (got.double() - want).abs() - U[q.dtype] * bound
    assert bool((err <= 1e-7).all()), float(err.max())
    return got


LENGTHS = {"mixed": [0, 1, 15, 16, 17, 63, 64, 65, 129, 300], "one": [1], "empty": [0, 0, 0], "long": [5000], "two": [2000, 7]}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 32, 80, 256])
@pytest.mark.parametrize("Hk,G", [(1, 1), (2, 3), (4, 8), (1, 9), (2, 16), (1, 33)])
@pytest.mark.parametrize("name,page_size", [("mixed", 16), ("mixed", 5), ("one", 1), ("empty", 32), ("long", 128), ("two", 64)])
def test_decode(dtype, D, Hk, G, name, page_size):
    lengths = LENGTHS[name]
    cache = _cache_of(lengths, page_size, Hk, D, dtype, seed=D + G)
    q = torch.randn(len(lengths), Hk * G, D, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    got = _check_decode(q, cache, lengths)
    for i, n in enumerate(lengths):
        if n == 0:
            assert not bool(got[i].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_peaked_scores_and_scales(dtype):
    """Scores far apart (one key takes all), equal ones, and a negative and a zero scale."""
    lengths = [700, 33, 5]
    cache = _cache_of(lengths, 16, 2, 64, dtype, stale=float("inf"))
    q = torch.randn(3, 8, 64, device="cuda").to(dtype)
    for scale in (4.0, 0.0, -0.125):
        _check_decode(q, cache, lengths, scale)


def test_decode_layouts_and_misaligned_queries():
    lengths = [100, 31, 64]
    for layout in ("heads", "tokens"):
        cache = _cache_of(lengths, 16, 2, 64, torch.bfloat16, layout=layout)
        wide = torch.randn(3, 24, 64, device="cuda").bfloat16()
        _check_decode(wide[:, 4:12], cache, lengths)
        _check_decode(wide.view(-1)[1:1 + 3 * 8 * 64].view(3, 8, 64), cache, lengths)
        _check_decode(wide[:, :1].expand(3, 8, 64), cache, lengths)


def test_decode_many_sequences_and_an_uneven_split():
    rng = random.Random(0)
    lengths = [rng.choice([0, 1, rng.randint(1, 400)]) for _ in range(321)] + [9000]
    cache = _cache_of(lengths, 16, 1, 64, torch.float16)
    _check_decode(torch.randn(322, 4, 64, device="cuda").half(), cache, lengths)


def test_decode_offsets_beyond_32_bits():
    """A pool of 2^31 elements and more; the pages in use lie at its end."""
    from nitrix_b200.nn import PagedCache

    page, Hk, D = 16, 2, 64
    pool = (1 << 31) // (page * Hk * D) + 50
    pages = torch.zeros(pool, Hk, page, D, dtype=torch.bfloat16, device="cuda")
    pages[-40:].normal_()
    table = torch.arange(pool - 1, pool - 36, -1, dtype=torch.int32, device="cuda")[None]
    n = torch.tensor([35 * page - 3], dtype=torch.int32, device="cuda")
    z = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = PagedCache(pages, pages, table, n, torch.zeros(pool, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), z)
    _check_decode(torch.randn(1, 8, D, device="cuda").bfloat16(), cache, [35 * page - 3])


def test_pages_beyond_32_bits():
    """Append, fork and compact in a pool of more than 2^31 elements, at its end."""
    from nitrix_b200.nn import PagedCache, cache_append, cache_compact, cache_fork

    page, Hk, D = 16, 2, 64
    pool = (1 << 31) // (page * Hk * D) + 100
    k_pages = torch.zeros(pool, Hk, page, D, dtype=torch.float16, device="cuda")
    ints = dict(dtype=torch.int32, device="cuda")
    order = torch.arange(pool - 1, -1, -1, **ints)
    cache = PagedCache(k_pages, torch.zeros_like(k_pages), torch.full((2, 8), -1, **ints), torch.zeros(2, **ints), order,
                       torch.tensor([0, pool], **ints), torch.zeros(1, **ints))
    k = torch.randn(70, Hk, D, device="cuda").half()
    cache = cache_append(cache, k, -k, torch.tensor([0, 37, 70], **ints))
    assert cache.table[:, :3].tolist() == [[pool - 1, pool - 2, pool - 3], [pool - 4, pool - 5, pool - 6]]

    def held(c, row, n):
        t = torch.arange(n, device="cuda")
        where = c.table[row].long()[t // page], slice(None), t % page
        return c.k_pages[where], c.v_pages[where]
    for c in (cache, cache_fork(cache, torch.tensor([1, 1, 0], **ints))):
        parents = [0, 1] if c.lengths.shape[0] == 2 else [1, 1, 0]
        packed = cache_compact(c)
        assert int(packed.table.max()) < 10
        for row, parent in enumerate(parents):
            want = k[:37] if parent == 0 else k[37:]
            for state in (c, packed):
                got = held(state, row, want.shape[0])
                assert torch.equal(got[0], want) and torch.equal(got[1], -want)


def test_decode_is_the_same_every_time():
    from nitrix_b200.nn import decode_attention

    lengths = [3000, 1, 777]
    cache = _cache_of(lengths, 16, 4, 128, torch.bfloat16)
    q = torch.randn(3, 16, 128, device="cuda").bfloat16()
    first = decode_attention(q, cache)
    for _ in range(5):
        assert torch.equal(decode_attention(q, cache), first)


def test_a_generation_step_in_a_graph():
    """Append and attention captured once, replayed with other tokens; lengths move on the device."""
    from nitrix_b200.nn import cache_append, decode_attention, paged_cache

    cache = paged_cache(64, 4, 2, 64, sequences=3, max_length=40, dtype=torch.bfloat16)
    k, v = (torch.randn(3, 2, 64, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(3, 4, 64, device="cuda").bfloat16()
    offsets = torch.arange(4, device="cuda").int()

    def step():
        after = cache_append(cache, k, v, offsets)
        out = decode_attention(q, after)
        cache.lengths.copy_(after.lengths)
        cache.free_range.copy_(after.free_range)
        return out
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(2, 12):
        for t in (k, v, q):
            t.copy_(torch.randn_like(t))
        graph.replay()
        torch.cuda.synchronize()
        assert cache.lengths.tolist() == [n] * 3
        want, bound = O.decode(q, cache.k_pages, cache.v_pages, cache.table, [n] * 3, 0.125)
        assert bool(((out.double() - want).abs() <= U[torch.bfloat16] * bound + 1e-7).all())


def test_refusals():
    from nitrix_b200.nn import cache_append, cache_compact, cache_fork, cache_free, decode_attention, paged_cache

    cache = paged_cache(8, 4, 2, 64, sequences=3, max_length=16)
    k = torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    offsets = torch.arange(4, device="cuda").int()
    q = torch.zeros(3, 4, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="positive"):
        paged_cache(0, 4, 2, 64, sequences=3, max_length=16)
    with pytest.raises(TypeError, match="k and v"):
        cache_append(cache, k.float(), k, offsets)
    with pytest.raises(ValueError, match="k and v"):
        cache_append(cache, k[:, :1], k, offsets)
    with pytest.raises(ValueError, match="offsets"):
        cache_append(cache, k, k, offsets[:3])
    with pytest.raises(TypeError, match="offsets"):
        cache_append(cache, k, k, offsets.long())
    with pytest.raises(TypeError, match="table"):
        cache_append(cache._replace(table=cache.table.cpu()), k, k, offsets)
    with pytest.raises(ValueError, match="table"):
        cache_append(cache._replace(table=cache.table.t().contiguous().t()), k, k, offsets)
    with pytest.raises(ValueError, match="lengths"):
        cache_compact(cache._replace(lengths=cache.lengths[:2]))
    with pytest.raises(ValueError, match="free_pages"):
        cache_compact(cache._replace(free_pages=cache.free_pages[:4]))
    with pytest.raises(TypeError, match="parents"):
        cache_fork(cache, torch.zeros(3, device="cuda"))
    with pytest.raises(TypeError, match="bool"):
        cache_free(cache, torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="finished"):
        cache_free(cache, torch.zeros(4, dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError, match="unit stride"):
        cache_compact(cache._replace(k_pages=cache.k_pages.transpose(2, 3).contiguous().transpose(2, 3)))
    with pytest.raises(ValueError, match="one shape"):
        cache_compact(cache._replace(v_pages=cache.v_pages[:4]))
    with pytest.raises(RuntimeError, match="16-byte"):
        odd = torch.zeros(8 * 2 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(8, 2, 4, 64)
        cache_compact(cache._replace(k_pages=odd))
    with pytest.raises(ValueError, match="q must be"):
        decode_attention(q[:, :3], cache)
    with pytest.raises(ValueError, match="q must be"):
        decode_attention(q[:2], cache)
    with pytest.raises(TypeError, match="q must be"):
        decode_attention(q.half(), cache)
    with pytest.raises(NotImplementedError, match="differentiable"):
        decode_attention(q.clone().requires_grad_(True), cache)
    with pytest.raises(RuntimeError, match="at most 256"):
        wide = paged_cache(2, 4, 1, 264, sequences=1, max_length=4)
        decode_attention(torch.zeros(1, 1, 264, device="cuda", dtype=torch.bfloat16), wide)
    assert cache_fork(cache, torch.zeros(0, dtype=torch.int32, device="cuda")).lengths.shape == (0,)


def test_refusals_of_pages():
    """Pools that no kernel may see: on the host, pages without a head or a slot."""
    from nitrix_b200.nn import PagedCache, cache_append, cache_compact, cache_fork, decode_attention, paged_cache

    cache = paged_cache(8, 4, 2, 64, sequences=3, max_length=16)
    k = torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    offsets = torch.arange(4, device="cuda").int()
    q = torch.zeros(3, 4, 64, device="cuda", dtype=torch.bfloat16)
    calls = [lambda c, k=k: cache_append(c, k, k, offsets), lambda c: cache_fork(c, offsets[:3]), cache_compact,
             lambda c: decode_attention(q, c)]
    host = PagedCache(*(t.cpu() for t in cache))
    for call in calls:
        with pytest.raises(TypeError, match="CUDA tensor"):
            call(host)
    for empty in (cache.k_pages[:, :0], cache.k_pages[:, :, :0]):
        for call in (lambda c: cache_append(c, k[:, :empty.shape[1]], k[:, :empty.shape[1]], offsets), *calls[1:]):
            with pytest.raises(ValueError, match="a token at least"):
                call(cache._replace(k_pages=empty, v_pages=empty))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 80, 256])
@pytest.mark.parametrize("G", [1, 4, 16])
def test_decode_an_infinity_in_the_last_value(dtype, D, G):
    """It reaches the element it stands in, as an infinity, and no other."""
    from nitrix_b200.nn import decode_attention

    lengths = [1, 5, 16, 33, 100, 700]
    cache = _cache_of(lengths, 16, 2, D, dtype, seed=D + G)
    q = torch.randn(len(lengths), 2 * G, D, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    want, bound = O.decode(q, cache.k_pages, cache.v_pages, cache.table, lengths, D ** -0.5)
    for i, n in enumerate(lengths):
        page, slot = cache.table[i, (n - 1) // 16].long(), (n - 1) % 16
        cache.v_pages[page, :, slot, 3] = float("inf")
        cache.v_pages[page, :, slot, 17] = -float("inf")
    got = decode_attention(q, cache).double()
    assert bool((got[..., 3] == float("inf")).all()) and bool((got[..., 17] == -float("inf")).all())
    rest = [d for d in range(D) if d not in (3, 17)]
    assert float(((got - want).abs() - U[dtype] * bound)[..., rest].max()) <= 1e-7


def test_offsets_that_leave_the_new_tokens():
    """Offsets that end behind ``k`` and ``v``, begin before them or descend: lengths and pages are those of what was stored."""
    from nitrix_b200.nn import cache_append

    def start():
        pair = Pair(20, 4, 3, 4)
        pair.append([5, 6, 7])
        return pair

    tokens = [100, 101, 102, 103, 104, 105]
    k = torch.tensor(tokens, dtype=torch.float32, device="cuda")[:, None, None].expand(6, 2, 8) + 0
    for offsets, stored, missing in (([0, 2, 4, 9], [tokens[:2], tokens[2:4], tokens[4:]], 3),
                                     ([0, 2, 40, 50], [tokens[:2], tokens[2:], []], 44),
                                     ([-4, 1, 2, 3], [tokens[:1], tokens[1:2], tokens[2:3]], 4),
                                     ([7, 8, 9, 2 ** 31 - 1], [[], [], []], 2 ** 31 - 8),
                                     ([0, 9, 2, 6], [[], [], []], 6),
                                     ([3, 2, 2, 1], [[], [], []], 6)):
        pair = start()
        pages = pair.cache.k_pages.clone()
        pair.cache = cache_append(pair.cache, k, -k, torch.tensor(offsets, dtype=torch.int32, device="cuda"))
        pair.model.append(stored)
        pair.model.shortfall += missing
        pair.check()
        if not any(stored):
            assert torch.equal(pair.cache.k_pages.nan_to_num(-1.0), pages.nan_to_num(-1.0))


def test_lengths_at_the_end_of_32_bits():
    """A table of one page many times over: 2^31 tokens and more.  A sequence counts 2^31 - 256 of them at most."""
    from nitrix_b200.nn import PagedCache, cache_append, decode_attention

    page, most = 1 << 16, 2 ** 31 - 256
    ints = dict(dtype=torch.int32, device="cuda")
    table = torch.zeros(1, (1 << 15) + 4, **ints)
    z = torch.zeros(1, **ints)
    for dtype, D in ((torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 80)):
        k = torch.zeros(1, 1, page, D, dtype=dtype, device="cuda")
        v = torch.full_like(k, 3.0)
        for n in (2 ** 31 - 1, most, most - 63):
            cache = PagedCache(k, v, table, torch.tensor([n], **ints), z, torch.zeros(2, **ints), z)
            out = decode_attention(torch.ones(1, 1, D, dtype=dtype, device="cuda"), cache)
            assert bool(((out - 3).abs() < 0.02).all())
    more = torch.zeros(4, 1, 80, dtype=torch.bfloat16, device="cuda")
    cache = cache_append(cache._replace(lengths=torch.tensor([most - 3], **ints)), more, more, torch.tensor([0, 4], **ints))
    assert cache.lengths.tolist() == [most] and cache.shortfall.tolist() == [1]


def test_autograd_notices_that_pages_are_written():
    """The calls write their pools in place: a graph that has saved one is told so, as by torch's own in-place operations."""
    from nitrix_b200.nn import cache_append, cache_compact, cache_fork, cache_free, paged_cache

    cache = paged_cache(16, 4, 2, 64, sequences=3, max_length=16, dtype=torch.float32)
    k = torch.randn(6, 2, 64, device="cuda")
    offsets = torch.tensor([0, 2, 4, 6], dtype=torch.int32, device="cuda")
    calls = {"append": lambda c: cache_append(c, k, k, offsets),
             "fork": lambda c: cache_fork(c, torch.tensor([0, 0, 2], dtype=torch.int32, device="cuda")),
             "free": lambda c: cache_free(c, torch.tensor([True, False, False], device="cuda")), "compact": cache_compact}
    for name, call in calls.items():
        before = cache.k_pages._version, cache.v_pages._version, cache.table._version
        w = torch.ones((), device="cuda", requires_grad=True)
        y = (cache.k_pages * w).sum()
        after = call(cache)
        if name == "free":      # (which writes no page)
            y.backward()
        else:
            assert cache.k_pages._version > before[0] and cache.v_pages._version > before[1]
            assert (cache.table._version > before[2]) == (name == "append")
            with pytest.raises(RuntimeError, match="inplace"):
                y.backward()
        cache = after
    with torch.inference_mode():
        inside = paged_cache(16, 4, 2, 64, sequences=3, max_length=16, dtype=torch.float32)
        inside = cache_append(inside, k, k, offsets)
    assert cache_append(inside, k, k, offsets).lengths.tolist() == [4, 4, 4]      # (such tensors have no version)


def test_forks_frees_and_compactions_in_a_graph():
    """Captured once each, replayed with other parents, other finished rows and other lengths."""
    from nitrix_b200.nn import cache_compact, cache_fork, cache_free

    rng = random.Random(2)
    pair = Pair(64, 4, 6, 8, Hk=2, D=64, dtype=torch.float32)
    state = [t.clone() for t in pair.cache]      # what the graphs read; the pools are shared
    state[0], state[1] = pair.cache.k_pages, pair.cache.v_pages
    parents = torch.arange(6, dtype=torch.int32, device="cuda")
    finished = torch.zeros(6, dtype=torch.bool, device="cuda")
    held = type(pair.cache)(*state)
    calls = {"fork": lambda: cache_fork(held, parents), "free": lambda: cache_free(held, finished), "compact": lambda: cache_compact(held)}
    graphs = {}
    side = torch.cuda.Stream()
    for name, call in calls.items():
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = call()
        graphs[name] = graph, result
    for _ in range(20):
        pair.append([rng.choice([0, 1, 3, 5]) for _ in range(6)])
        what = rng.choice(list(calls))
        if what == "fork":
            chosen = [rng.randint(-1, 5) for _ in range(6)]
            parents.copy_(torch.tensor(chosen))
            pair.model.fork(chosen)
        elif what == "free":
            flags = [rng.random() < 0.4 for _ in range(6)]
            finished.copy_(torch.tensor(flags))
            pair.model.fork([-1 if f else i for i, f in enumerate(flags)])
        else:
            pair.model.compact()
        for to, now in zip(state[2:], pair.cache[2:]):
            to.copy_(now)
        graph, result = graphs[what]
        graph.replay()
        pair.cache = type(pair.cache)(pair.cache.k_pages, pair.cache.v_pages, *(t.clone() for t in result[2:]))
        torch.cuda.synchronize()
        pair.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [1e-20, 1e-34, 2e-38, 1e-38])
def test_decode_scales_near_the_end_of_fp32(dtype, scale):
    """The mean of the values."""
    lengths = [700, 33, 5]
    cache = _cache_of(lengths, 16, 2, 64, dtype)
    _check_decode(torch.randn(3, 8, 64, device="cuda").to(dtype), cache, lengths, scale)
