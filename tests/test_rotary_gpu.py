"""Rotary positions on the GPU against the rotation in 64 bits.

An element is x1 cos - x2 sin in fp32 from cosines good to 2e-7 (the phase is reduced in 64 bits, its fp32 remainder is off by
2^-24 of half a turn), so within 8e-7 (|x1| + |x2|) of the exact value; a 16-bit result is rounded once, by half an ulp.
"""
import pytest
import torch

from oracle import decoder_oracle as O

pytestmark = pytest.mark.gpu

HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def _close(got, x, want, dtype, pairs):
    spread = 8e-7 * 2 * x.double().abs().amax(-1, keepdim=True)
    bound = spread + HALF_ULP[dtype] * (want.abs() + spread) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() - bound).max())
    assert torch.equal(got[..., 2 * pairs:], x[..., 2 * pairs:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lead,H,Hk,D,sections", [
    ((1,), 1, 1, 64, (32,)), ((5,), 32, 8, 128, (64,)), ((300,), 4, 2, 128, (16, 24, 24)), ((3, 77), 6, 3, 64, (16,)),
    ((2, 2, 9), 2, 1, 256, (128,)), ((40,), 3, 3, 80, (13, 7)), ((33,), 5, 1, 20, (4, 0, 3)), ((0,), 2, 2, 64, (32,)),
    ((700,), 16, 16, 128, (64,)), ((6,), 300, 20, 64, (8, 8))])
def test_forward_and_gradient(dtype, interleaved, lead, H, Hk, D, sections):
    from nitrix_b200.nn import rotary_embedding, rotary_frequencies

    g = torch.Generator(device="cuda").manual_seed(D + H)
    q, k, gq, gk = (torch.randn(*lead, h, D, generator=g, device="cuda").to(dtype) for h in (H, Hk, H, Hk))
    freq = rotary_frequencies(sections, device="cuda")
    pos = torch.randint(-3, 200000, (*lead, len(sections)), generator=g, device="cuda").int()
    qg, kg = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    yq, yk = rotary_embedding(qg, kg, pos, freq, sections=sections, interleaved=interleaved)
    dq, dk = torch.autograd.grad([yq, yk], [qg, kg], [gq, gk])
    if q.numel() == 0:
        assert yq.shape == q.shape and dk.shape == k.shape
        return
    pairs = sum(sections)
    for x, y, grad, d in ((q, yq, gq, dq), (k, yk, gk, dk)):
        assert y.dtype == dtype and y.is_contiguous()
        _close(y.detach(), x, O.rotary(x, pos, freq, sections, interleaved), dtype, pairs)
        _close(d, grad, O.rotary(grad, pos, freq, sections, interleaved, inverse=True), dtype, pairs)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_positions_far_away_and_of_every_type(kind):
    from nitrix_b200.nn import rotary_embedding, rotary_frequencies

    x = torch.randn(64, 2, 64, device="cuda")
    pos = (torch.arange(64, device="cuda") * 16777216).to(kind)       # up to 2^30, exact in fp32
    if kind == torch.int64:
        pos = pos * 1024
    freq = rotary_frequencies((32,), device="cuda")
    y, none = rotary_embedding(x, None, pos, freq)
    assert none is None
    _close(y, x, O.rotary(x, pos[:, None], freq, (32,)), torch.float32, 32)


def test_gradient_against_differences():
    """The map is linear: <g, R(x + e) - R(x)> = <grad, e> up to fp32 rounding of the two sides (64 terms of size 1)."""
    from nitrix_b200.nn import rotary_embedding, rotary_frequencies

    g = torch.Generator(device="cuda").manual_seed(3)
    x, e, ct = (torch.randn(7, 3, 64, generator=g, device="cuda") for _ in range(3))
    freq, pos = rotary_frequencies((32,), device="cuda"), torch.arange(7, device="cuda").int()
    leaf = x.clone().requires_grad_(True)
    y, _ = rotary_embedding(leaf, None, pos, freq)
    grad, = torch.autograd.grad(y, leaf, ct)
    moved, _ = rotary_embedding(x + e, None, pos, freq)
    left = ((moved.double() - y.detach().double()) * ct.double()).sum()
    right = (grad.double() * e.double()).sum()
    assert abs(float(left - right)) < 1344 * 8 * 2.0 ** -23


def test_views_and_layouts():
    """Slices of one projection, a (batch, heads, length, D) buffer seen as tokens first, odd offsets and expanded rows give
    what dense operands give."""
    from nitrix_b200.nn import rotary_embedding, rotary_frequencies

    g = torch.Generator(device="cuda").manual_seed(4)
    freq, pos = rotary_frequencies((32,), device="cuda"), torch.arange(24, device="cuda").reshape(2, 12).int()
    qkv = torch.randn(2, 12, 12, 64, generator=g, device="cuda").bfloat16()
    heads_first = torch.randn(2, 3, 12, 64, generator=g, device="cuda").bfloat16()
    odd = torch.randn(2 * 12 * 3 * 64 + 1, generator=g, device="cuda").bfloat16()[1:].view(2, 12, 3, 64)
    expanded = torch.randn(2, 12, 1, 64, generator=g, device="cuda").bfloat16().expand(2, 12, 3, 64)
    backwards = torch.randn(2, 12, 64, 3, generator=g, device="cuda").bfloat16().transpose(2, 3)
    for a, b in ((qkv[:, :, :8], qkv[:, :, 8:10]), (heads_first.transpose(1, 2), odd), (expanded, backwards)):
        got = rotary_embedding(a, b, pos, freq)
        want = rotary_embedding(a.contiguous().clone(), b.contiguous().clone(), pos, freq)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_gradient_of_one_result_alone_and_an_expanded_cotangent():
    from nitrix_b200.nn import rotary_embedding, rotary_frequencies

    freq, pos = rotary_frequencies((32,), device="cuda"), torch.arange(9, device="cuda").int()
    q, k = (torch.randn(9, h, 64, device="cuda", requires_grad=True) for h in (4, 2))
    _, yk = rotary_embedding(q, k, pos, freq)
    yk.sum().backward()
    assert q.grad is None
    ones = torch.ones(9, 2, 64, device="cuda")
    _close(k.grad, ones, O.rotary(ones, pos[:, None], freq, (32,), inverse=True), torch.float32, 32)


def test_on_another_stream_and_in_a_graph():
    from nitrix_b200.nn import rotary_embedding, rotary_frequencies

    freq, pos = rotary_frequencies((32,), device="cuda"), torch.arange(50, device="cuda").int()
    x = torch.randn(50, 4, 64, device="cuda")
    want, _ = rotary_embedding(x, None, pos, freq)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = rotary_embedding(x, None, pos, freq)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again, _ = rotary_embedding(x, None, pos, freq)
    x.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, -want)


def test_refusals():
    from nitrix_b200.nn import rotary_embedding, rotary_frequencies

    q, freq = torch.randn(4, 2, 64, device="cuda"), rotary_frequencies((32,), device="cuda")
    pos = torch.arange(4, device="cuda").int()
    with pytest.raises(TypeError, match="CUDA tensor"):
        rotary_embedding(q.cpu(), None, pos, freq)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        rotary_embedding(q.double(), None, pos, freq)
    with pytest.raises(TypeError, match="positions"):
        rotary_embedding(q, None, pos.short(), freq)
    with pytest.raises(TypeError, match="positions"):
        rotary_embedding(q, None, pos.cpu(), freq)
    with pytest.raises(ValueError, match="positions"):
        rotary_embedding(q, None, pos[:3], freq)
    with pytest.raises(ValueError, match="positions"):
        rotary_embedding(q, None, pos, freq, sections=(16, 16))
    with pytest.raises(TypeError, match="frequencies"):
        rotary_embedding(q, None, pos, freq.double())
    with pytest.raises(ValueError, match="frequencies"):
        rotary_embedding(q, None, pos, freq, sections=(16,))
    with pytest.raises(ValueError, match="do not fit"):
        rotary_embedding(q, None, pos, rotary_frequencies((33,), device="cuda"))
    with pytest.raises(ValueError, match="axes"):
        rotary_embedding(q, None, pos, freq, sections=(4,) * 9)
    with pytest.raises(ValueError, match="k must be"):
        rotary_embedding(q, q[:3], pos, freq)
    with pytest.raises(TypeError, match="k must be"):
        rotary_embedding(q, q.half(), pos, freq)
    with pytest.raises(ValueError, match="not differentiable"):
        rotary_embedding(q, None, pos, freq.clone().requires_grad_(True))
    with pytest.raises(RuntimeError, match="at most 256"):
        wide = torch.randn(4, 2, 260, device="cuda")
        rotary_embedding(wide, None, pos, freq)
    with pytest.raises(ValueError):
        rotary_frequencies(())


def test_more_tokens_than_32_bits_count():
    from nitrix_b200.nn import rotary_embedding

    q = torch.zeros(1, 1, 8, device="cuda", dtype=torch.bfloat16).expand(2 ** 32 + 1, 1, 8)
    positions = torch.zeros(1, dtype=torch.int32, device="cuda").expand(2 ** 32 + 1)
    with pytest.raises(ValueError, match="32 bits"):
        rotary_embedding(q, None, positions, torch.ones(4, device="cuda"))


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_positions_around_the_first_that_fp32_does_not_hold(kind):
    """2^24 + 1 as an fp32 number is 2^24: one radian away at frequency 1."""
    from nitrix_b200.nn import rotary_embedding, rotary_frequencies

    n = 1 << 24
    pos = torch.tensor([n - 1, n, n + 1, n + 2, n + 3, -n - 1, -n, 1 - n], device="cuda").to(kind)
    x, ct = (torch.randn(8, 2, 64, device="cuda") for _ in range(2))
    freq = rotary_frequencies((32,), device="cuda")
    leaf = x.clone().requires_grad_(True)
    y, _ = rotary_embedding(leaf, None, pos, freq)
    _close(y.detach(), x, O.rotary(x, pos[:, None], freq, (32,)), torch.float32, 32)
    grad, = torch.autograd.grad(y, leaf, ct)
    _close(grad, ct, O.rotary(ct, pos[:, None], freq, (32,), inverse=True), torch.float32, 32)
