"""The root-mean-square norm on the GPU against 64 bits: forward, gradients, and the output in 8 bits.

Sums of rows and columns are fp32, of at most 80 terms one after the other and a tree of the rest, and every factor is rounded a few
times: F = 100 roundings of fp32 bound what they add up to, relative to the sums of magnitudes that the oracle gives.  Results are
rounded once to their type, half an ulp; e4m3 codes too, 2^-4 of their value or half of the smallest step.
"""
import pytest
import torch

from oracle import few_bits_oracle as O

pytestmark = pytest.mark.gpu

F = 100 * 2.0 ** -24
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TINY = 2.0 ** -25       # half of fp16's smallest step
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _operands(shape, dtype, residual=True, weight=True, seed=0, wide=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda").to(dtype)
    r = (3 * torch.randn(shape, generator=g, device="cuda")).to(dtype) if residual else None
    w = (1 + 0.3 * torch.randn(shape[-1], generator=g, device="cuda")) if weight else None
    return x, r, w if w is None or wide else w.to(dtype)


def _close(got, want, bound, name):
    err = (got.detach().double() - want.detach()).abs() - HALF[got.dtype] * want.detach().abs() - F * bound.detach() - TINY
    assert not bool(got.isnan().any()) and float(err.max()) <= 0, (name, float(err.max()))


def _run(shape, dtype, residual=True, weight=True, wide=False, eps=1e-6, seed=0):
    from nitrix_b200.nn import rms_norm

    x, r, w = _operands(shape, dtype, residual, weight, seed, wide)
    leaves = [t.requires_grad_(True) for t in (x, r, w) if t is not None]
    out = rms_norm(x, w, residual=r, eps=eps)
    y, h = (out, x) if r is None else out
    assert y.dtype == dtype and y.shape == x.shape and y.is_contiguous()
    assert torch.equal(h, O.stream_sum(x, r))
    want, _, _ = O.rms_norm(h.detach(), w, eps)
    _close(y, want, want.abs(), "y")
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    dy, dh = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
    grads = torch.autograd.grad([y] if r is None else [y, h], leaves, [dy] if r is None else [dy, dh])
    dx, dx_bound, dw, dw_bound = O.rms_norm_grads(h.detach(), w, eps, dy, None if r is None else dh)
    _close(grads[0], dx, dx_bound, "dx")
    if r is not None:
        assert torch.equal(grads[0], grads[1])
    if w is not None:
        assert grads[-1].dtype == w.dtype
        _close(grads[-1], dw, dw_bound, "dw")
    return y.detach()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [1, 7, 8, 31, 32, 100, 256, 264, 1000, 1024, 1001, 2048, 2056, 4096, 5120, 8192, 8200])
def test_every_width(C, dtype):
    _run((3, 13, C), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [8191, 8193, 16384, 16392, 16400, 20001])
def test_rows_too_wide_to_be_held(C, dtype):
    _run((5, C), dtype)
    _run((70, C), dtype, residual=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [0, 1, 2, 9, 1500, 2001])
def test_numbers_of_rows(rows, dtype):
    for C in (64, 512, 2048, 257):
        if rows:
            _run((rows, C), dtype, seed=rows)


@pytest.mark.parametrize("residual,weight,wide", [(False, True, False), (False, False, False), (True, False, False), (True, True, True), (False, True, True)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_operands_that_are_left_out_and_fp32_weights(dtype, residual, weight, wide):
    for C in (96, 1001, 4096):
        _run((40, C), dtype, residual, weight, wide, eps=1e-3)


def test_no_rows_and_no_axes_in_front():
    from nitrix_b200.nn import rms_norm, rms_norm_quantized

    x = torch.zeros(0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y, h = rms_norm(x, w, residual=x)
    dx, dw = torch.autograd.grad([y, h], [x, w], [torch.zeros_like(y), torch.zeros_like(h)])
    assert y.shape == h.shape == dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))
    codes, scales = rms_norm_quantized(x.detach())
    assert codes.shape == (0, 64) and scales.shape == (0, 1)
    _run((129,), torch.bfloat16)


def test_rows_of_zeros_and_of_extreme_numbers():
    from nitrix_b200.nn import rms_norm

    for dtype in DTYPES:
        x = torch.zeros(4, 64, device="cuda", dtype=dtype)
        x[1] = 6e4
        x[2] = 1e-4
        want, _, _ = O.rms_norm(x, None, 1e-6)
        _close(rms_norm(x), want, want.abs(), dtype)
        x[3, 5] = float("nan")
        assert bool(rms_norm(x)[3].isnan().all()) and not bool(rms_norm(x)[:3].isnan().any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    """Strided, expanded and misaligned operands give what dense ones give."""
    from nitrix_b200.nn import rms_norm

    wide = torch.randn(6, 5, 300, device="cuda").to(dtype)
    for x in (wide[..., 3:259], wide[:, ::2, :256], wide.transpose(0, 1)[..., :256], wide[:1, :, :256].expand(6, 5, 256),
              wide.view(-1)[1:1 + 20 * 256].view(20, 256)):
        w = torch.randn(257, device="cuda").to(dtype)[1:]
        leaves = [t.detach().requires_grad_(True) for t in (x, w)]
        dense = [t.detach().clone().contiguous().requires_grad_(True) for t in (x, w)]
        outs = [rms_norm(a, b, residual=a) for a, b in (leaves, dense)]
        assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
        dy = torch.randn(x.shape[::-1], device="cuda").to(dtype).permute(*range(x.dim() - 1, -1, -1))
        got, want = (torch.autograd.grad(o[0], l, dy) for o, l in zip(outs, (leaves, dense)))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradients_of_either_output_alone_and_the_same_every_time():
    from nitrix_b200.nn import rms_norm

    x, r, w = (t.requires_grad_(True) for t in _operands((700, 1024), torch.bfloat16))
    y, h = rms_norm(x, w, residual=r)
    dy, dh = torch.randn_like(y), torch.randn_like(h)
    dx, dr, dw = torch.autograd.grad(y, [x, r, w], dy, retain_graph=True)
    want, bound, want_dw, dw_bound = O.rms_norm_grads(h.detach(), w, 1e-6, dy)
    _close(dx, want, bound, "dx")
    _close(dw, want_dw, dw_bound, "dw")
    for _ in range(3):
        again = torch.autograd.grad(y, [x, r, w], dy, retain_graph=True)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dr) and torch.equal(again[2], dw)
    dx, dr = torch.autograd.grad(h, [x, r], dh, retain_graph=True)
    assert torch.equal(dx, dh) and torch.equal(dr, dh)
    assert torch.autograd.grad(h, [w], dh, allow_unused=True) == (None,)


def test_gradients_against_differences():
    from nitrix_b200.nn import rms_norm

    x, r, w = (t.requires_grad_(True) for t in _operands((4, 40), torch.float32))
    dy, dh = torch.randn(4, 40, device="cuda"), torch.randn(4, 40, device="cuda")
    grads = torch.autograd.grad(rms_norm(x, w, residual=r), [x, r, w], [dy, dh])
    for i, leaf in enumerate((x, r, w)):
        way = torch.randn_like(leaf)
        step = 2.0 ** -10

        def value(sign):
            ops = [t.detach().double() + (sign * step * way.double() if j == i else 0) for j, t in enumerate((x, r, w))]
            y, _, _ = O.rms_norm(ops[0] + ops[1], ops[2], 1e-6)
            return float((y * dy.double()).sum() + ((ops[0] + ops[1]) * dh.double()).sum())
        want = (value(1) - value(-1)) / (2 * step)
        # (the differences' own error is of the order of step^2)
        assert abs(float((grads[i].double() * way.double()).sum()) - want) <= 1e-4 * (1 + abs(want))


# ---- 8 bits ------------------------------------------------------------------------------------------------------------------
def _check_eight(x, r, w, group, eps=1e-6):
    from nitrix_b200.nn import rms_norm_quantized

    out = rms_norm_quantized(x, w, residual=r, eps=eps, group_size=group)
    codes, scales = out[:2]
    h = O.stream_sum(x, r)
    if r is not None:
        assert torch.equal(out[2], h)
    y, _, _ = O.rms_norm(h, w, eps)
    want = O.scales_of(y, group)
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == x.shape
    assert scales.dtype == torch.float32 and scales.shape == (*x.shape[:-1], x.shape[-1] // group if group else 1)
    assert float(((scales.double() - want).abs() / want).max()) <= F
    z = y / want.repeat_interleave(group or x.shape[-1], -1)
    # half a step is at most 2^-4 of a value, or 2^-10; fp32's own errors move the value before it is rounded
    err = (codes.double() - z).abs() - (2.0 ** -4 * z.abs()).clamp(min=2.0 ** -10) * (1 + 1e-3) - F * z.abs()
    assert float(err.max()) <= 0, float(err.max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [1, 30, 64, 257, 1024, 4096, 8192, 8194, 16512, 17001])
def test_eight_bits_of_rows(C, dtype):
    _check_eight(*_operands((9, C), dtype), None)
    _check_eight(*_operands((2, 3, C), dtype, residual=False, wide=True, seed=1), None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group,C", [(32, 32), (32, 96), (64, 64), (64, 4096), (128, 128), (128, 384), (128, 8192), (64, 16512), (32, 2080)])
def test_eight_bits_of_groups(group, C, dtype):
    x, r, w = _operands((11, C), dtype, wide=C == 384)
    x[2], r[2] = 0, 0
    _check_eight(x, r, w, group)
    _check_eight(x.view(-1)[:-C].view(10, C), None, None, group)
    odd = torch.empty(10 * C + 1, dtype=dtype, device="cuda")[1:].view(10, C).copy_(x[:10])      # (not on a 16-byte boundary)
    _check_eight(odd, r[:10], w, group)


def test_eight_bits_of_zeros_and_of_what_is_not_finite():
    from nitrix_b200.nn import rms_norm_quantized

    x = torch.randn(4, 256, device="cuda").bfloat16()
    x[1] = 0
    x[2, 7], x[3, 200] = float("nan"), float("inf")
    for group in (None, 32):
        codes, scales = rms_norm_quantized(x, group_size=group)
        assert not bool(codes[1].float().any()) and bool((scales[1] > 0).all())
        assert not bool(codes[0].float().isnan().any())
        assert bool(codes[2].float().isnan().all())
        # (an infinity: the factor of its row is zero, so it is a NaN and the others are zeros)
        spoiled = codes[3].float().isnan()
        assert bool(spoiled.all()) if group is None else bool(spoiled[192:224].all()) and not bool(codes[3, :192].float().any())


# ---- as it is called -----------------------------------------------------------------------------------------------------------
def test_another_stream_and_a_graph():
    from nitrix_b200.nn import rms_norm, rms_norm_quantized

    x, r, w = _operands((300, 512), torch.float16)
    want = rms_norm(x, w, residual=r), rms_norm_quantized(x, w, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rms_norm(x, w, residual=r), rms_norm_quantized(x, w, residual=r)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = rms_norm(x, w, residual=r), rms_norm_quantized(x, w, residual=r)
    x.copy_(x.flip(0)), r.copy_(r.flip(0))
    graph.replay()
    for a, b, c in zip([*want[0], *want[1]], [*got[0], *got[1]], [*held[0], *held[1]]):
        assert torch.equal(a.float(), b.float()) and torch.equal(a.float().flip(0), c.float())


def test_a_training_step_in_a_graph():
    from nitrix_b200.nn import rms_norm

    x, r, w = (t.requires_grad_(True) for t in _operands((300, 520), torch.bfloat16))
    dy, dh = torch.randn(300, 520, device="cuda").bfloat16(), torch.randn(300, 520, device="cuda").bfloat16()

    def step():
        return torch.autograd.grad(rms_norm(x, w, residual=r), [x, r, w], [dy, dh])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(2):
        with torch.no_grad():
            x.normal_(), dy.normal_()
        graph.replay()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_what_has_no_rule_is_refused():
    from nitrix_b200.nn import rms_norm, rms_norm_quantized

    x, r, w = _operands((5, 64), torch.float32)
    dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
    for call in (lambda: rms_norm(dual(x), w), lambda: rms_norm(x, dual(w)), lambda: rms_norm(x, w, residual=dual(r)), lambda: rms_norm_quantized(dual(x))):
        with pytest.raises(NotImplementedError, match="forward-mode"), torch.autograd.forward_ad.dual_level():
            call()
    for ops in ((x.clone().requires_grad_(True), w, r), (x, w.clone().requires_grad_(True), r), (x, w, r.clone().requires_grad_(True))):
        with pytest.raises(NotImplementedError, match="differentiable"):
            rms_norm_quantized(ops[0], ops[1], residual=ops[2])
        with torch.no_grad():
            rms_norm_quantized(ops[0], ops[1], residual=ops[2])
    leaf = x.clone().requires_grad_(True)
    y = rms_norm(leaf * 1, w)
    (gx,) = torch.autograd.grad(y.square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), leaf)
    z = leaf * 1
    y = rms_norm(z, w)
    z.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    y, h = rms_norm(leaf, w, residual=r)
    h.add_(1)       # (the sum is what the backward pass reads)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


def test_gradients_through_hooks_and_of_some_operands():
    from nitrix_b200.nn import rms_norm

    leaves = [t.requires_grad_(True) for t in _operands((50, 96), torch.float32)]
    f = lambda x, r, w: sum(t.square().sum() for t in rms_norm(x, w, residual=r))
    want = torch.autograd.grad(f(*leaves), leaves)
    for i, leaf in enumerate(leaves):
        only = [t if j == i else t.detach() for j, t in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(f(*only), [leaf])[0], want[i])
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        y = f(*leaves)
    for a, b in zip(torch.autograd.grad(y, leaves), want):
        assert torch.equal(a, b)


def test_refusals():
    from nitrix_b200.nn import rms_norm, rms_norm_quantized

    x, r, w = _operands((5, 64), torch.bfloat16)
    for f in (rms_norm, rms_norm_quantized):
        with pytest.raises(TypeError, match="x must be"):
            f(x.double())
        with pytest.raises(TypeError, match="x must be"):
            f(x.cpu())
        with pytest.raises(TypeError, match="residual"):
            f(x, residual=r.float())
        with pytest.raises(TypeError, match="residual"):
            f(x, residual=r.cpu())
        with pytest.raises(ValueError, match="residual"):
            f(x, residual=r[:4])
        with pytest.raises(TypeError, match="weight"):
            f(x, w.half())
        with pytest.raises(TypeError, match="weight"):
            f(x, w.cpu())
        with pytest.raises(ValueError, match="weight"):
            f(x, w[:32])
        with pytest.raises(ValueError, match="channel"):
            f(x[:, :0])
        with pytest.raises(ValueError, match="channel"):
            f(x[0, 0])
    for group in (16, 48, 0, -32):
        with pytest.raises(ValueError, match="group_size"):
            rms_norm_quantized(x, group_size=group)
    with pytest.raises(ValueError, match="group_size"):
        rms_norm_quantized(x[:, :48].contiguous(), group_size=32)


def test_more_than_2_to_the_31_elements():
    """The last rows of tensors whose offsets leave 32 bits are those of the rows alone."""
    from nitrix_b200.nn import rms_norm, rms_norm_quantized

    rows, C = 2 ** 31 // 8192 + 40, 8192
    x = torch.empty(rows, C, dtype=torch.bfloat16, device="cuda")
    x[-50:].normal_()
    w = torch.randn(C, device="cuda").bfloat16()
    few = x[-50:].clone()
    y = rms_norm(x, w)
    assert torch.equal(y[-50:], rms_norm(few, w))
    del y
    for group in (None, 128):
        codes, scales = rms_norm_quantized(x, w, group_size=group)
        want = rms_norm_quantized(few, w, group_size=group)
        assert torch.equal(codes[-50:].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scales[-50:], want[1])
        del codes, scales
    x[:-50] = 0
    a, b = x.requires_grad_(True), few.requires_grad_(True)
    dy = torch.zeros_like(x)
    dy[-50:].normal_()
    (da,), (db,) = torch.autograd.grad(rms_norm(a, w), [a], dy), torch.autograd.grad(rms_norm(b, w), [b], dy[-50:])
    assert torch.equal(da[-50:], db) and not bool(da[:1000].any())


@pytest.mark.parametrize("dtype,C", [(torch.float32, 1 << 29), (torch.bfloat16, 1 << 30)])
def test_rows_of_2_to_the_31_bytes(dtype, C):
    """Of ones of either sign, whose squares' sum is exact: the norm is the row times (1 + eps)^-1/2, within 2^-20."""
    from nitrix_b200.nn import rms_norm

    x = torch.empty(1, C, dtype=dtype, device="cuda").bernoulli_(0.5).mul_(2).sub_(1)
    y = rms_norm(x)
    assert float((y - x).abs().max()) <= 2.0 ** -20 + HALF[dtype]
    del y
    with pytest.raises(ValueError, match="2\\^30"):
        rms_norm(torch.empty(0, (1 << 30) + 1, dtype=dtype, device="cuda"))
    if dtype == torch.float32:
        # a gradient in the last 8 columns alone: mean(g n) is 8 / C, which is what the other columns get, against their sign
        dy = torch.zeros_like(x)
        dy[:, -8:] = x[:, -8:]
        x.requires_grad_(True)
        (dx,) = torch.autograd.grad(rms_norm(x), [x], dy)
        dx *= x.detach()
        assert float((dx[:, :-8] * (C / 8) + 1).abs().max()) < 2.0 ** -18 and float((dx[:, -8:] - 1).abs().max()) < 2.0 ** -18
