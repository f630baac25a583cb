"""Attention over packed sequences on the GPU against 64 bits, forward and gradients.

16-bit operands: probabilities, their gradients and the results are each rounded once to the operand type, the row sums of the
backward come from a rounded output, all else is fp32.  The oracle returns with every value the sum that such a relative error
multiplies, so the bound is u times that sum, u half an ulp, doubled for the fp32 parts (and exponentials good to 1e-4 relative,
which 16-bit forwards may use: below a tenth of an fp16 ulp's half).  fp32: 1e-5 of the same sums.
"""
import random

import pytest
import torch

from oracle import decoder_oracle as O

pytestmark = pytest.mark.gpu

U = {t: torch.finfo(t).eps for t in (torch.bfloat16, torch.float16)} | {torch.float32: 1e-5}


def _offsets(lengths):
    return torch.tensor([0, *lengths]).cumsum(0).int().cuda()


def _inputs(lengths_q, lengths_k, H, Hk, D, dtype, seed=0, extra=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tq, tk = sum(lengths_q) + extra, sum(lengths_k) + extra
    q, k, v, dout = (torch.randn(t, h, D, generator=g, device="cuda").to(dtype) for t, h in ((tq, H), (tk, Hk), (tk, Hk), (tq, H)))
    return q, k, v, dout


def _check(q, k, v, dout, lengths_q, lengths_k, causal=True, scale=None, backend="auto", offsets=None):
    from nitrix_b200 import _cabi
    from nitrix_b200.nn import packed_attention

    dtype = q.dtype
    oq = _offsets(lengths_q)
    ok = None if lengths_k is lengths_q else _offsets(lengths_k)
    with torch.no_grad():
        plain = packed_attention(q, k, v, oq, offsets_k=ok, causal=causal, scale=scale, backend=backend)
    leaves = [t.detach().clone(memory_format=torch.preserve_format).requires_grad_(True) if t.is_contiguous() else t.detach().requires_grad_(True)
              for t in (q, k, v)]
    out = packed_attention(*leaves, oq, offsets_k=ok, causal=causal, scale=scale, backend=backend)
    grads = torch.autograd.grad(out, leaves, dout)
    torch.cuda.synchronize()
    assert _cabi.lib().nb200_device_status(0) == 0
    assert torch.equal(plain, out.detach())
    want = O.packed(q, k, v, lengths_q, lengths_k, q.shape[-1] ** -0.5 if scale is None else scale, causal, dout)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)):
        value, bound = want[name]
        assert got.dtype == dtype and got.shape == value.shape
        err = (got.double() - value).abs() - U[dtype] * bound
        assert bool((err <= 1e-6).all()), (name, float(err.max()))
    return out.detach(), grads


SHAPES = {
    "one token": [1],
    "tile edges": [63, 64, 65, 127, 128, 129],
    "empty ones": [0, 5, 0, 0, 200, 1, 0],
    "one longer": [700],
    "many short": [3, 1, 17, 9, 2, 31, 16, 8, 40, 5, 1, 1, 12],
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 40, 256])
@pytest.mark.parametrize("Hk,G", [(1, 1), (2, 4), (1, 3), (2, 8), (1, 16)])
@pytest.mark.parametrize("name", SHAPES)
def test_causal(dtype, D, Hk, G, name, monkeypatch):
    monkeypatch.setenv("NITRIX_SILENCE_FALLBACK", "1")
    lengths = SHAPES[name]
    _check(*_inputs(lengths, lengths, Hk * G, Hk, D, dtype, seed=D + G), lengths, lengths)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths_q,lengths_k", [
    ([5, 100, 64], [300, 100, 0]), ([200, 1, 33], [7, 129, 256]), ([0, 40, 130], [50, 0, 129]), ([300], [128]), ([1, 1, 1], [257, 1, 64])])
def test_keys_of_other_lengths(dtype, D, causal, lengths_q, lengths_k, monkeypatch):
    """Fewer keys than queries leave the first queries without any under causal: zeros, and no gradient."""
    monkeypatch.setenv("NITRIX_SILENCE_FALLBACK", "1")
    out, grads = _check(*_inputs(lengths_q, lengths_k, 8, 2, D, dtype), lengths_q, lengths_k, causal)
    at = 0
    for lq, lk in zip(lengths_q, lengths_k):
        blind = lq if lk == 0 else (max(lq - lk, 0) if causal else 0)
        assert not bool(out[at:at + blind].any()) and not bool(grads[0][at:at + blind].any())
        at += lq


@pytest.mark.parametrize("D,Hk,G", [(64, 1, 5), (128, 1, 7), (64, 2, 32), (128, 1, 64), (64, 1, 65), (128, 3, 2), (64, 1, 128)])
def test_group_sizes(D, Hk, G, monkeypatch):
    monkeypatch.setenv("NITRIX_SILENCE_FALLBACK", "1")
    lengths = [70, 3, 141]
    _check(*_inputs(lengths, lengths, Hk * G, Hk, D, torch.bfloat16), lengths, lengths)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [1.5, 0.0, -0.3])
def test_scales(dtype, scale, monkeypatch):
    monkeypatch.setenv("NITRIX_SILENCE_FALLBACK", "1")
    lengths = [150, 20]
    _check(*_inputs(lengths, lengths, 4, 2, 64, dtype), lengths, lengths, scale=scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
def test_a_sequence_does_not_see_its_neighbours(dtype, D, monkeypatch):
    """NaN and infinities in every other sequence, and in the tokens behind the last, stay there -- in the gradients too."""
    from nitrix_b200.nn import packed_attention

    monkeypatch.setenv("NITRIX_SILENCE_FALLBACK", "1")
    lengths = [37, 130, 64, 200, 1, 90]
    q, k, v, dout = _inputs(lengths, lengths, 6, 2, D, dtype, extra=11)
    spans, at = [], 0
    for n in lengths:
        spans.append(slice(at, at + n))
        at += n
    clean = [i for i in range(len(lengths)) if i % 2 == 0]

    def run(*operands):
        leaves = [t.clone().requires_grad_(True) for t in operands[:3]]
        out = packed_attention(*leaves, _offsets(lengths))
        return [out.detach(), *torch.autograd.grad(out, leaves, operands[3])]
    want = run(q, k, v, dout)
    for bad in (float("nan"), float("inf")):
        dirty = [t.clone() for t in (q, k, v, dout)]
        for t in dirty:
            for i, s in enumerate(spans):
                if i not in clean:
                    t[s] = bad
            t[at:] = bad
        got = run(*dirty)
        for a, b in zip(got, want):
            for i in clean:
                # (the sums of dq are made in no fixed order)
                assert bool(torch.isfinite(a[spans[i]]).all())
                assert float((a[spans[i]].double() - b[spans[i]].double()).abs().max()) <= 2 * U[dtype] * float(b[spans[i]].double().abs().max())
            assert not bool(a[at:].any())


def test_views_of_one_projection_and_expanded_cotangents():
    lengths = [100, 29, 300]
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn(429, 12, 64, generator=g, device="cuda").bfloat16()
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    dout = torch.randn(429, 8, 64, generator=g, device="cuda").bfloat16()
    _check(q, k, v, dout, lengths, lengths)
    _check(q, k, v, torch.ones((), device="cuda", dtype=torch.bfloat16).expand(429, 8, 64), lengths, lengths)
    odd = torch.randn(429 * 8 * 64 + 1, generator=g, device="cuda").bfloat16()[1:].view(429, 8, 64)
    _check(odd, k, v, dout, lengths, lengths)


def test_gradients_against_differences():
    """fp32, central differences along random directions: truncation is O(h^2) of third derivatives of order one; with h = 1e-2
    the fp32 noise of a sum of 23 040 outputs over 2 h stays below 2e-2, as does h^2."""
    from nitrix_b200.nn import packed_attention

    lengths = [33, 60, 27]
    q, k, v, dout = _inputs(lengths, lengths, 3, 1, 64, torch.float32)
    off = _offsets(lengths)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(packed_attention(*leaves, off, backend="cuda-simt"), leaves, dout)
    g = torch.Generator(device="cuda").manual_seed(9)
    for i in range(3):
        e = torch.randn(leaves[i].shape, generator=g, device="cuda")
        e /= e.norm()
        h = 1e-2

        def f(sign):
            ops = [q, k, v]
            ops[i] = ops[i] + sign * h * e
            return (packed_attention(*ops, off, backend="cuda-simt").double() * dout.double()).sum()
        assert abs(float((f(1) - f(-1)) / (2 * h) - (grads[i].double() * e.double()).sum())) < 2e-2


def test_fp16_gradients_of_long_sequences():
    """Thousands of keys: P and dS are small, where fp16 has fewer digits.  The roundings of dS and of the results are 2^-11 at
    most, 2.1e-4 in the root mean square of values spread over a binade, and independent; a third one of that size stands for
    delta's and P's: sqrt(3) * 2.1e-4 in the 2-norm."""
    from nitrix_b200.nn import packed_attention

    lengths = [6000]
    q, k, v, dout = _inputs(lengths, lengths, 2, 1, 64, torch.float16)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(packed_attention(*leaves, _offsets(lengths)), leaves, dout)
    want = O.packed(q, k, v, lengths, lengths, 0.125, True, dout)
    for name, got in zip(("dq", "dk", "dv"), grads):
        value = want[name][0]
        assert float((got.double() - value).norm() / value.norm()) < 3.7e-4, name


def test_fp16_gradients_whose_products_leave_fp16():
    """dout and v so large that dS itself would overflow; the gradients do not."""
    lengths = [300, 40]
    q, k, v, dout = _inputs(lengths, lengths, 4, 2, 128, torch.float16)
    _check(q * 0.01, k * 0.01, v * 30, dout * 1000, lengths, lengths)
    _check(q * 0.01, k * 0.01, v * 0, dout * 0, lengths, lengths)


def test_families_and_reproducibility(monkeypatch):
    import nitrix_b200
    from nitrix_b200.backend import NitrixBackendError, NitrixBackendFallback, reset_fallback_state
    from nitrix_b200.nn import packed_attention

    lengths = [90, 40]
    q, k, v, dout = _inputs(lengths, lengths, 4, 2, 64, torch.bfloat16)
    off = _offsets(lengths)

    def run():
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        out = packed_attention(*leaves, off)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    with nitrix_b200.reproducible():
        first = run()
        for _ in range(3):
            for a, b in zip(run(), first):
                assert torch.equal(a, b)
    reset_fallback_state()
    with pytest.warns(NitrixBackendFallback, match="packed_attention"):
        packed_attention(q.float(), k.float(), v.float(), off)
    monkeypatch.setenv("NITRIX_STRICT_BACKEND", "1")
    with pytest.raises(NitrixBackendError):
        packed_attention(q.float(), k.float(), v.float(), off)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_random_batches(dtype):
    rng = random.Random(5)
    for _ in range(25):
        D, Hk, G = rng.choice([64, 128]), rng.choice([1, 2, 3]), rng.choice([1, 2, 3, 4, 5, 8, 12])
        n = rng.randint(1, 9)
        lq = [rng.choice([0, 1, rng.randint(1, 30), rng.randint(1, 400)]) for _ in range(n)]
        lk = lq if rng.random() < 0.5 else [rng.choice([0, 1, rng.randint(1, 30), rng.randint(1, 400)]) for _ in range(n)]
        _check(*_inputs(lq, lk, Hk * G, Hk, D, dtype, seed=n), lq, lk, rng.random() < 0.7)


def test_streams_and_graphs():
    from nitrix_b200.nn import packed_attention

    lengths = [130, 20, 55]
    q, k, v, _ = _inputs(lengths, lengths, 4, 2, 128, torch.bfloat16)
    off = _offsets(lengths)
    want = packed_attention(q, k, v, off)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = packed_attention(q, k, v, off)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = packed_attention(q, k, v, off)
    other = [20, 130, 55]
    off.copy_(_offsets(other))        # other lengths, the same graph
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, packed_attention(q, k, v, _offsets(other)))


def test_offsets_that_make_no_sense_stay_in_bounds():
    """Offsets that run backwards, overlap or leave the tensors: no access outside, no hang; what comes out means nothing."""
    from nitrix_b200 import _cabi
    from nitrix_b200.nn import packed_attention

    q, k, v, dout = _inputs([300], [300], 6, 2, 64, torch.bfloat16)
    for bad in ([0, 300] * 40, [0, 900, -5, 20, 7, 300], [300, 0, 300, 0, 300], [-(1 << 30), 1 << 30, 0, 1 << 30], [50, 60]):
        off = torch.tensor(bad, dtype=torch.int32, device="cuda")
        for backend in ("auto", "cuda-simt"):
            leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
            torch.autograd.grad(packed_attention(*leaves, off, backend=backend), leaves, dout)
    torch.cuda.synchronize()
    assert _cabi.lib().nb200_device_status(0) == 0


def test_refusals():
    from nitrix_b200.nn import packed_attention

    q, k, v, _ = _inputs([10], [10], 4, 2, 64, torch.bfloat16)
    off = _offsets([10])
    with pytest.raises(TypeError, match="CUDA tensor"):
        packed_attention(q.cpu(), k, v, off)
    with pytest.raises(TypeError, match="k and v"):
        packed_attention(q, k.half(), v, off)
    with pytest.raises(ValueError, match="head dim"):
        packed_attention(q, k, v[:, :1], off)
    with pytest.raises(ValueError, match="multiple"):
        packed_attention(q[:, :3], k, v, off)
    with pytest.raises(TypeError, match="offsets"):
        packed_attention(q, k, v, off.long())
    with pytest.raises(ValueError, match="offsets"):
        packed_attention(q, k, v, off[None])
    with pytest.raises(ValueError, match="offsets_k"):
        packed_attention(q[:9], k, v, off)
    with pytest.raises(ValueError, match="offsets_k"):
        packed_attention(q, k, v, off, offsets_k=_offsets([5, 5]))
    with pytest.raises(RuntimeError, match="at most 256"):
        packed_attention(*(t.repeat(1, 1, 5) for t in (q, k, v)), off, backend="cuda-simt")
    empty = packed_attention(q[:0], k[:0], v[:0], _offsets([0, 0]))
    assert empty.shape == (0, 4, 64)
    assert not bool(packed_attention(q, k, v, _offsets([]), backend="cuda-simt").any())


def test_more_tokens_than_32_bits_count():
    from nitrix_b200.nn import packed_attention

    q = torch.zeros(1, 1, 64, device="cuda", dtype=torch.bfloat16)
    many = q.expand(2 ** 32 + 1, 1, 64)
    with pytest.raises(ValueError, match="32 bits"):
        packed_attention(many, many, many, _offsets([1]))


LONG = {
    "one": [300],
    "edges": [128, 127, 129, 256],
    "empty and short ones": [0, 700, 1, 64, 65, 0, 500],
    "two tiles and a row": [257, 130],
}


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hk,G", [(1, 1), (2, 3), (1, 4), (1, 16), (1, 128), (3, 1)])
@pytest.mark.parametrize("name", LONG)
def test_fp32_on_the_tensor_cores(D, Hk, G, name):
    """Three bf16 numbers per operand: what is left out of a product is below 2^-20 of it, and the accumulators, emptied every
    other step, truncate 48 times by 2^-24: 4e-6 of the sums of either product, within the 1e-5 of fp32."""
    from nitrix_b200 import _cabi

    lengths = LONG[name]
    before = _cabi.lib().nb200_launch_count()
    _check(*_inputs(lengths, lengths, Hk * G, Hk, D, torch.float32, seed=D + G), lengths, lengths)
    assert _cabi.lib().nb200_launch_count() > before


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths_q,lengths_k", [
    ([5, 100, 64], [300, 500, 0]), ([200, 1, 33], [137, 129, 256]), ([400, 300], [300, 5]), ([1, 90], [777, 64]), ([64], [4000])])
def test_fp32_keys_of_other_lengths(D, causal, lengths_q, lengths_k):
    out, grads = _check(*_inputs(lengths_q, lengths_k, 8, 2, D, torch.float32), lengths_q, lengths_k, causal)
    at = 0
    for lq, lk in zip(lengths_q, lengths_k):
        blind = lq if lk == 0 else (max(lq - lk, 0) if causal else 0)
        assert not bool(out[at:at + blind].any()) and not bool(grads[0][at:at + blind].any())
        at += lq


def test_fp32_more_blocks_than_a_wave_and_strides():
    """Two query tiles per CTA; views of one projection, operands that are not 16-byte aligned, tokens behind the last offset."""
    from nitrix_b200.nn import packed_attention

    lengths = [1000, 30, 900, 0, 300, 129]
    g = torch.Generator(device="cuda").manual_seed(4)
    n = sum(lengths)
    qkv = torch.randn(n, 24, 64, generator=g, device="cuda")
    q, k, v = qkv[:, :16], qkv[:, 16:20], qkv[:, 20:]
    dout = torch.randn(n, 16, 64, generator=g, device="cuda")
    _check(q, k, v, dout, lengths, lengths)
    _check(q, k, v, dout, lengths, lengths, scale=-0.2)
    odd = torch.randn(n * 16 * 64 + 1, generator=g, device="cuda")[1:].view(n, 16, 64)
    _check(odd, k, v, dout, lengths, lengths, causal=False)
    with torch.no_grad():
        more = [torch.cat([t, torch.full((700, *t.shape[1:]), float("nan"), device="cuda")]) for t in (q, k, v)]
        out = packed_attention(*more, _offsets(lengths))
        assert torch.equal(out[:n], packed_attention(q, k, v, _offsets(lengths)))
        assert not bool(out[n:].any())


def test_fp32_neighbours_and_magnitudes():
    """NaN and infinities of a neighbour stay there; operands of 1e-18 and 1e18 keep their digits."""
    from nitrix_b200.nn import packed_attention

    lengths = [200, 131, 300, 77]
    q, k, v, dout = _inputs(lengths, lengths, 4, 2, 128, torch.float32)
    off = _offsets(lengths)
    with torch.no_grad():
        want = packed_attention(q, k, v, off)
        for bad in (float("nan"), float("inf")):
            dirty = [t.clone() for t in (q, k, v)]
            for t in dirty:
                t[200:331] = bad
                t[631:] = bad
            got = packed_attention(*dirty, off)
            assert torch.equal(got[:200], want[:200]) and torch.equal(got[331:631], want[331:631])
        big = packed_attention(q * 2.0 ** 60, k * 2.0 ** -60, v * 2.0 ** -60, off)
        assert torch.equal(big, want * 2.0 ** -60)


@pytest.mark.parametrize("Hk,G,lengths", [(4, 16, [600, 0, 300, 200]), (8, 64, [300, 257]), (3, 5, [700, 31, 129]), (16, 4, [1, 270])])
def test_fp32_gradients_of_groups(Hk, G, lengths):
    """Groups whose rows fill the tiles and groups that leave some unused; the same bits every time."""
    operands = _inputs(lengths, lengths, Hk * G, Hk, 64, torch.float32, seed=G)
    out, grads = _check(*operands, lengths, lengths)
    again, more = _check(*operands, lengths, lengths)
    assert torch.equal(out, again) and all(torch.equal(a, b) for a, b in zip(grads, more))


def test_fp32_gradients_on_the_tensor_cores_against_differences():
    """As above; 55 680 outputs that are good to 2^-20 each leave 2^-20 sqrt(55 680) / (2 h) = 1e-2 at most."""
    from nitrix_b200.nn import packed_attention

    lengths = [140, 150]
    q, k, v, dout = _inputs(lengths, lengths, 3, 1, 64, torch.float32)
    off = _offsets(lengths)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(packed_attention(*leaves, off), leaves, dout)
    g = torch.Generator(device="cuda").manual_seed(9)
    for i in range(3):
        e = torch.randn(leaves[i].shape, generator=g, device="cuda")
        e /= e.norm()
        h = 1e-2

        def f(sign):
            ops = [q, k, v]
            ops[i] = ops[i] + sign * h * e
            return (packed_attention(*ops, off).double() * dout.double()).sum()
        assert abs(float((f(1) - f(-1)) / (2 * h) - (grads[i].double() * e.double()).sum())) < 2e-2


@pytest.mark.parametrize("dtype,D,backend", [
    (torch.bfloat16, 64, "auto"), (torch.float16, 128, "auto"), (torch.float32, 64, "auto"), (torch.float32, 128, "auto"),
    (torch.bfloat16, 64, "cuda-simt"), (torch.float32, 40, "cuda-simt"), (torch.float16, 256, "cuda-simt")])
@pytest.mark.parametrize("lead_q,lead_k", [(37, 37), (5, 130), (200, 0)])
def test_tokens_before_the_first_offset(dtype, D, backend, lead_q, lead_k, monkeypatch):
    """Sequences cut out of a longer batch: what lies before the first offset belongs to none of them, as what lies behind the
    last: zeros, in the gradients too, whatever its operands hold."""
    from nitrix_b200.nn import packed_attention

    monkeypatch.setenv("NITRIX_SILENCE_FALLBACK", "1")
    lengths_q, lengths_k = [300, 0, 140], [260, 31, 190]
    nq, nk = sum(lengths_q), sum(lengths_k)
    q, k, v, dout = _inputs([lead_q + nq + 21], [lead_k + nk + 21], 4, 2, D, dtype)
    rows, keys = slice(lead_q, lead_q + nq), slice(lead_k, lead_k + nk)
    for t, s in ((q, rows), (k, keys), (v, keys), (dout, rows)):
        t[:s.start] = float("nan")
        t[s.stop:] = float("nan")
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    stale = [torch.full_like(t, float("nan")) for t in (q, q, k, v) for _ in range(3)]      # what the results are given to write on
    del stale
    out = packed_attention(*leaves, _offsets(lengths_q) + lead_q, offsets_k=_offsets(lengths_k) + lead_k, backend=backend)
    stale = [torch.full_like(t, float("nan")) for t in (q, k, v) for _ in range(3)]
    del stale
    grads = torch.autograd.grad(out, leaves, dout)
    want = O.packed(q[rows], k[keys], v[keys], lengths_q, lengths_k, D ** -0.5, True, dout[rows])
    for name, got, s in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads), (rows, rows, keys, keys)):
        assert not bool(got[:s.start].any()) and not bool(got[s.stop:].any()), name
        value, bound = want[name]
        assert float(((got[s].double() - value).abs() - U[dtype] * bound).max()) <= 1e-6, name


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [3e2, 6e4])
def test_fp16_gradients_beside_large_numbers(D, size):
    """Numbers of any size in neighbouring sequences, and in rows of no sequence, take no digits from the gradients of the others."""
    from nitrix_b200.nn import packed_attention

    lengths, lead, tail = [200, 150, 33, 1, 100], 19, 70
    n = lead + sum(lengths)
    q, k, v, dout = _inputs([n + tail], [n + tail], 6, 2, D, torch.float16)
    dout *= 1e-3
    spans, at = [], lead
    for length in lengths:
        spans.append(slice(at, at + length))
        at += length
    dirty = [slice(0, lead), spans[1], spans[3], slice(n, n + tail)]
    for s in dirty:
        v[s] = size
        dout[s] = -size
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(packed_attention(*leaves, _offsets(lengths) + lead), leaves, dout)
    for i in (0, 2, 4):
        s = spans[i]
        want = O.packed(q[s], k[s], v[s], [lengths[i]], [lengths[i]], D ** -0.5, True, dout[s])
        for name, got in zip(("dq", "dk", "dv"), grads):
            value, bound = want[name]
            assert float(((got[s].double() - value).abs() - U[torch.float16] * bound).max()) <= 1e-6, (i, name)


@pytest.mark.parametrize("D", [64, 128])
def test_fp16_gradients_where_the_row_statistics_leave_fp16(D):
    """Scores, sums of out * dout and 1 / scale so large that no few fp16 numbers hold a row's lse / scale or delta: the gradients
    are as good as elsewhere."""
    lengths = [150, 20, 300]
    q, k, v, dout = _inputs(lengths, lengths, 4, 2, D, torch.float16)
    _check(q, k, v * 0 + 200, dout * 0 + 1000, lengths, lengths)         # delta: 1.3e7 and 2.6e7
    for scale in (1e-5, 1e-7, 1e-9):
        _check(q, k, v, dout, lengths, lengths, scale=scale)
    _check(q * 5000, k * 5000, v, dout, lengths, lengths, scale=1e-8)    # scores of 1e9 before the scale, of 10 after it
    _check(q * 5000, k * 5000, v, dout, lengths, lengths, scale=1e-8, causal=False)


@pytest.mark.parametrize("D", [64, 128])
def test_fp16_gradients_of_equal_scores_of_millions(D):
    """All scores 2e7 before the scale (1e7 at head dim 64): lse is 1.3e6 to 2.6e6, where fp32 steps by 1/8 and 1/4.  Two roundings
    of it are a factor of 2^(1/4) in a row's probabilities at most, 0.19 of them."""
    from nitrix_b200.nn import packed_attention

    lengths = [150, 40]
    q, k, v, dout = _inputs(lengths, lengths, 4, 2, D, torch.float16)
    q, k = q * 0 + 400, k * 0 + 400
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = packed_attention(*leaves, _offsets(lengths))
    grads = torch.autograd.grad(out, leaves, dout)
    want = O.packed(q, k, v, lengths, lengths, D ** -0.5, True, dout)
    for name, got, u in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads), (0.0, 0.19, 0.19, 0.19)):
        value, bound = want[name]
        assert float(((got.double() - value).abs() - (u + U[torch.float16]) * bound).max()) <= 1e-6, name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_near_the_end_of_fp32(dtype, monkeypatch):
    monkeypatch.setenv("NITRIX_SILENCE_FALLBACK", "1")
    lengths = [150, 20]
    for scale in (1e-25, 1e-34, 2e-38, 1e-38):
        _check(*_inputs(lengths, lengths, 4, 2, 64, dtype), lengths, lengths, scale=scale)


def test_what_falls_back_is_told_once_per_head_layout(monkeypatch):
    """Batches differ in their number of tokens every time: that is no new problem to tell of, nor to remember."""
    from nitrix_b200 import backend
    from nitrix_b200.nn import packed_attention

    backend.reset_fallback_state()
    with pytest.warns(backend.NitrixBackendFallback, match="head dim 64 or 128"):
        for n in (20, 21, 22, 40):
            packed_attention(*_inputs([n], [n], 4, 2, 64, torch.float32)[:3], _offsets([n]))
    assert len(backend._warned_keys) == 1
    packed_attention(*_inputs([20], [20], 8, 2, 64, torch.float32)[:3], _offsets([20]))
    assert len(backend._warned_keys) == 2
    backend.reset_fallback_state()


def test_empty_batches_fall_back_to_nothing(monkeypatch):
    from nitrix_b200.nn import packed_attention

    monkeypatch.setenv("NITRIX_STRICT_BACKEND", "1")
    q, k, v, dout = _inputs([10], [10], 4, 2, 64, torch.bfloat16)
    assert packed_attention(q[:0], k[:0], v[:0], _offsets([0, 0])).shape == (0, 4, 64)
    assert packed_attention(q[:0], k, v, _offsets([0]), offsets_k=_offsets([10])).shape == (0, 4, 64)
    leaves = [t.clone().requires_grad_(True) for t in (q, k[:0], v[:0])]
    out = packed_attention(*leaves, _offsets([4, 6]), offsets_k=_offsets([0, 0]))
    assert not bool(out.any())
    assert not bool(torch.autograd.grad(out, leaves, dout)[0].any())
    assert not bool(packed_attention(q, k, v, _offsets([])).any())


def test_a_gradient_that_leaves_the_tensor_cores_is_told(monkeypatch):
    """fp32 of head dim 128: the forward pass stays on them, its gradient does not."""
    from nitrix_b200 import backend
    from nitrix_b200.nn import packed_attention

    q, k, v, dout = _inputs([300], [300], 4, 2, 128, torch.float32)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    off = _offsets([300])
    backend.reset_fallback_state()
    with pytest.warns(backend.NitrixBackendFallback, match="gradients"):
        packed_attention(*leaves, off)
    monkeypatch.setenv("NITRIX_STRICT_BACKEND", "1")
    with pytest.raises(backend.NitrixBackendError, match="gradients"):
        packed_attention(*leaves, off)
    packed_attention(q, k, v, off)                                       # no gradient is asked for
    with torch.no_grad():
        packed_attention(*leaves, off)
    for dtype, D in ((torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)):
        packed_attention(*(t[..., :D].to(dtype).detach().requires_grad_(True) for t in leaves), off)
    backend.reset_fallback_state()


@pytest.mark.parametrize("dtype,D,backend", [
    (torch.bfloat16, 64, "auto"), (torch.float16, 64, "auto"), (torch.bfloat16, 128, "auto"), (torch.float16, 128, "auto"),
    (torch.float32, 64, "auto"), (torch.float32, 128, "auto"), (torch.bfloat16, 64, "cuda-simt"), (torch.float32, 40, "cuda-simt"),
    (torch.float16, 256, "cuda-simt")])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_a_query_without_keys_holds_reaches_no_gradient(dtype, D, backend, bad, monkeypatch):
    """More queries than keys under causal: the first see none, and neither their row of q nor that of dout takes part."""
    from nitrix_b200.nn import packed_attention

    monkeypatch.setenv("NITRIX_SILENCE_FALLBACK", "1")
    lengths_q, lengths_k = [300, 33, 0, 140, 200], [260, 190, 20, 11, 199]
    q, k, v, dout = _inputs(lengths_q, lengths_k, 6, 2, D, dtype)
    at = 0
    clean = [t.clone() for t in (q, dout)]
    for lq, lk in zip(lengths_q, lengths_k):
        blind = slice(at, at + max(lq - lk, 0))
        q[blind], dout[blind] = bad, bad
        clean[0][blind], clean[1][blind] = 0, 0
        at += lq
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = packed_attention(*leaves, _offsets(lengths_q), offsets_k=_offsets(lengths_k), backend=backend)
    grads = torch.autograd.grad(out, leaves, dout)
    want = O.packed(clean[0], k, v, lengths_q, lengths_k, D ** -0.5, True, clean[1])
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)):
        value, bound = want[name]
        assert float(((got.double() - value).abs() - U[dtype] * bound).max()) <= 1e-6, name
