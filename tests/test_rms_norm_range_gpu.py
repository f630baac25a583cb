"""The root-mean-square norm at the ends of its range: long rows, many rows, numbers whose squares leave fp32.

The bounds are those of the other tests of the norm: sums of at most 80 fp32 terms one after the other (longer ones are folded into
64 bits every 64 terms) and a tree of the rest, F = 100 roundings of fp32 relative to the sums of magnitudes, half an ulp of the result.
"""
import pytest
import torch

from oracle import few_bits_oracle as O

pytestmark = pytest.mark.gpu

F = 100 * 2.0 ** -24
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TINY = 2.0 ** -25       # half of fp16's smallest step
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _close(got, want, bound, name):
    err = (got.detach().double() - want.detach()).abs() - HALF[got.dtype] * want.detach().abs() - F * bound.detach() - TINY
    assert not bool(got.isnan().any()) and float(err.max()) <= 0, (name, float(err.max()))


# ---- long rows -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("C", [1 << 20, (1 << 20) + 1, 1 << 24])
@pytest.mark.parametrize("dtype", DTYPES)
def test_long_rows(C, dtype):
    """Rows of equal numbers, whose roundings all go one way where they are added one by one, and random ones.  (The scales of the output in
    8 bits show 16-bit rows' factors in fp32.)"""
    from nitrix_b200.nn import rms_norm, rms_norm_quantized

    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(3, C, dtype=dtype, device="cuda")
    x[0], x[1] = 0.3, 1.7
    x[2].normal_(generator=g)
    want, _, _ = O.rms_norm(x, None, 1e-6)
    _close(rms_norm(x), want, want.abs(), "y")
    scales = rms_norm_quantized(x)[1]
    exact = O.scales_of(want, None)
    assert float(((scales.double() - exact).abs() / exact).max()) <= F
    dy = x.flip(0).contiguous()
    for leaf, cot in ((x, dy), (x, torch.full_like(x, 0.3))):
        leaf = leaf.detach().requires_grad_(True)
        (dx,) = torch.autograd.grad(rms_norm(leaf), leaf, cot)
        want_dx, bound, _, _ = O.rms_norm_grads(leaf.detach(), None, 1e-6, cot)
        _close(dx, want_dx, bound, "dx")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("C", [32768, 32776, 32896, 65536])
def test_16_bit_rows_at_and_beyond_what_is_held(C, dtype):
    """32768 channels are held in the forward, more are read twice, by words; with and without a residual, weights of either type."""
    from nitrix_b200.nn import rms_norm, rms_norm_quantized

    g = torch.Generator(device="cuda").manual_seed(C)
    x, r = (torch.randn(5, C, generator=g, device="cuda").to(dtype) for _ in range(2))
    dy, dh = (torch.randn(5, C, generator=g, device="cuda").to(dtype) for _ in range(2))
    for residual, w in ((r, torch.randn(C, generator=g, device="cuda")), (None, torch.randn(C, generator=g, device="cuda").to(dtype)), (r, None)):
        leaves = [t.detach().requires_grad_(True) for t in (x, residual, w) if t is not None]
        out = rms_norm(leaves[0], None if w is None else leaves[-1], residual=None if residual is None else leaves[1])
        y, h = (out, x) if residual is None else (out[0], out[1].detach())
        assert torch.equal(h, O.stream_sum(x, residual))
        want, _, _ = O.rms_norm(h, w, 1e-6)
        _close(y, want, want.abs(), "y")
        grads = torch.autograd.grad(y if residual is None else out, leaves, dy if residual is None else [dy, dh])
        dx, dx_bound, dw, dw_bound = O.rms_norm_grads(h, w, 1e-6, dy, None if residual is None else dh)
        _close(grads[0], dx, dx_bound, "dx")
        if w is not None:
            _close(grads[-1], dw, dw_bound, "dw")
        for group in (None, 32, 64, 128) if C % 128 == 0 else (None,):
            codes, scales, *rest = rms_norm_quantized(x, w, residual=residual, group_size=group)
            assert not rest or torch.equal(rest[0], h)
            exact = O.scales_of(want, group)
            assert float(((scales.double() - exact).abs() / exact).max()) <= F
            z = want / exact.repeat_interleave(group or C, -1)
            err = (codes.double() - z).abs() - (2.0 ** -4 * z.abs()).clamp(min=2.0 ** -10) * (1 + 1e-3) - F * z.abs()
            assert float(err.max()) <= 0, float(err.max())


# ---- many rows -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,rows,C", [
    (torch.float32, 1 << 24, 32), (torch.float32, 1 << 24, 7), (torch.bfloat16, 1 << 24, 64), (torch.bfloat16, 1 << 21, 1000),
    (torch.float16, 1 << 20, 2048), (torch.bfloat16, 1 << 18, 8193), (torch.bfloat16, 1 << 18, 16400)])
def test_gradients_of_weights_over_many_rows(dtype, rows, C):
    """Of rows that are all alike: dw is their number times one term, of which 256 at most are added one after the other, 8 groups of rows and
    32 CTAs' sums in fp32 again, the rest in 64 bits and a tree: 305 roundings."""
    from nitrix_b200.nn import rms_norm

    x, w = torch.full((rows, C), 1.7, dtype=dtype, device="cuda"), torch.ones(C, device="cuda", requires_grad=True)
    y = rms_norm(x, w)
    dy = torch.full_like(x, 0.3)
    dy[:, 1::2] = -1.1
    (dw,) = torch.autograd.grad(y, w, dy)
    n = O.rms_norm(x[:1], None, 1e-6)[0]
    want = rows * (n * dy[:1].double())[0]
    assert float(((dw.double() - want).abs() / want.abs()).max()) <= 305 * 2.0 ** -24


@pytest.mark.parametrize("dtype,C", [(torch.float32, 32), (torch.bfloat16, 2056), (torch.float16, 129)])
@pytest.mark.parametrize("more", [0, 1, 5003])
def test_rows_about_a_launch_s_end(dtype, C, more):
    """The backward takes 256 rows a thread in a launch; every row behind has its gradient, and its part of dw, all the same."""
    from nitrix_b200.nn import rms_norm

    sms = torch.cuda.get_device_properties(0).multi_processor_count
    rows = 256 * sms * {32: 4 * 8, 2056: 3, 129: 4 * 4}[C] + more      # (CTAs of an SM times rows of a CTA)
    g = torch.Generator(device="cuda").manual_seed(more)
    x, r, dy, dh = (torch.randn(rows, C, generator=g, device="cuda").to(dtype) for _ in range(4))
    w = torch.randn(C, generator=g, device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, r, w)]
    y, h = rms_norm(x, w, residual=r)
    dx, dr, dw = torch.autograd.grad([y, h], leaves, [dy, dh])
    again = torch.autograd.grad(rms_norm(x, w, residual=r), leaves, [dy, dh])
    assert torch.equal(dw, again[2]) and torch.equal(dx, again[0]) and torch.equal(dx, dr)
    h, w = h.detach(), w.detach()
    want_dw, bound_dw = torch.zeros(C, dtype=torch.float64, device="cuda"), torch.zeros(C, dtype=torch.float64, device="cuda")
    for at in range(0, rows, 1 << 18):
        part = slice(at, at + (1 << 18))
        want, bound, terms, terms_bound = O.rms_norm_grads(h[part], w, 1e-6, dy[part], dh[part])
        _close(dx[part], want, bound, "dx")
        want_dw += terms
        bound_dw += terms_bound
    assert float(((dw.double() - want_dw).abs() - 305 * 2.0 ** -24 * bound_dw).max()) <= 0


# ---- numbers whose squares leave fp32 ----------------------------------------------------------------------------------------------
WIDTHS = [64, 257, 1000, 4096, 8193, 16400, 40000]


def _rows(C, dtype, residual):
    """Rows of one size each, from that whose squares' sum leaves fp32 up to the largest numbers; one that stands alone; a usual one."""
    g = torch.Generator(device="cuda").manual_seed(C)
    size = torch.tensor([1e18, 1e19, 1.8e19, 1e25, 1e30, 4e37, 1.0], device="cuda")
    x = (torch.rand(7, C, generator=g, device="cuda") + 0.5) * size[:, None]
    x[:, ::3] *= -1
    x = torch.cat([x, torch.randn(2, C, generator=g, device="cuda"), torch.full((1, C), 3.0e38, device="cuda")])
    x[7, C // 2] = -3e38
    x = x.to(dtype)
    r = (x.float() * torch.rand(10, C, generator=g, device="cuda") * 0.1).to(dtype) if residual else None
    return x, r


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("residual", [False, True])
def test_squares_that_leave_fp32(C, dtype, residual):
    from nitrix_b200.nn import rms_norm

    x, r = _rows(C, dtype, residual)
    w = torch.linspace(0.5, 1.5, C, device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, r, w) if t is not None]
    out = rms_norm(x, w, residual=r)
    y, h = out if residual else (out, x)
    h = h.detach()
    assert torch.equal(h, O.stream_sum(x.detach(), None if r is None else r.detach())) and bool(h.isfinite().all())
    want, _, _ = O.rms_norm(h, w.detach(), 1e-6)
    _close(y, want, want.abs(), "y")
    dy = torch.randn(x.shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    grads = torch.autograd.grad(y, leaves, dy)
    dx, dx_bound, dw, dw_bound = O.rms_norm_grads(h, w.detach(), 1e-6, dy)
    _close(grads[0], dx, dx_bound, "dx")
    _close(grads[-1], dw, dw_bound, "dw")


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_squares_that_vanish_from_fp32(C, dtype):
    """With an eps that leaves them be."""
    from nitrix_b200.nn import rms_norm

    g = torch.Generator(device="cuda").manual_seed(C)
    size = torch.tensor([1e-15, 1e-18, 1e-20, 1e-25, 1e-30, 1.0], device="cuda")
    x = (torch.randn(6, C, generator=g, device="cuda") * size[:, None]).to(dtype)
    w = torch.linspace(0.5, 1.5, C, device="cuda")
    dy = torch.randn(x.shape, generator=g, device="cuda").to(dtype)
    for eps in (0.0, 1e-38):
        leaves = [x.detach().requires_grad_(True), w.detach().requires_grad_(True)]
        y = rms_norm(*leaves, eps=eps)
        eps = float(torch.tensor(eps))
        want, _, _ = O.rms_norm(x, w, eps)
        _close(y, want, want.abs(), "y")
        grads = torch.autograd.grad(y, leaves, dy)
        dx, dx_bound, dw, dw_bound = O.rms_norm_grads(x, w, eps, dy)
        _close(grads[0], dx, dx_bound, "dx")
        _close(grads[1], dw, dw_bound, "dw")


@pytest.mark.parametrize("C", [128, 4096, 8192, 40064, 1001, 17001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_eight_bits_of_squares_that_leave_fp32(C, dtype):
    from nitrix_b200.nn import rms_norm_quantized

    x, r = _rows(C, dtype, True)
    h = O.stream_sum(x, r)
    y, _, _ = O.rms_norm(h, None, 1e-6)
    for group in (None, 32, 128) if C % 128 == 0 else (None,):
        codes, scales, got = rms_norm_quantized(x, residual=r, group_size=group)
        assert torch.equal(got, h)
        want = O.scales_of(y, group)
        assert float(((scales.double() - want).abs() / want).max()) <= F
        z = y / want.repeat_interleave(group or C, -1)
        err = (codes.double() - z).abs() - (2.0 ** -4 * z.abs()).clamp(min=2.0 ** -10) * (1 + 1e-3) - F * z.abs()
        assert float(err.max()) <= 0, float(err.max())


@pytest.mark.parametrize("C", [64, 4096, 20000])
def test_infinities_and_nan_beside_large_numbers(C):
    """An infinity has a NaN, the others of its row zeros; a NaN spoils its row; other rows are what they are."""
    from nitrix_b200.nn import rms_norm

    x = torch.full((6, C), 1e30, device="cuda").bfloat16()
    x[1, 5], x[3, C - 1], x[4, 0] = float("inf"), -float("inf"), float("nan")
    y = rms_norm(x).float()
    for row, at in ((1, 5), (3, C - 1)):
        spoiled = torch.zeros(C, dtype=torch.bool, device="cuda")
        spoiled[at] = True
        assert torch.equal(y[row].isnan(), spoiled) and not bool(y[row][~spoiled].any())
    assert bool(y[4].isnan().all())
    assert bool((y[[0, 2, 5]] == 1).all())


@pytest.mark.parametrize("C", [40, 520, 1024, 4096, 8192, 1001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_rows_among_many_change_no_other(C, dtype):
    from nitrix_b200.nn import rms_norm, rms_norm_quantized

    g = torch.Generator(device="cuda").manual_seed(0)
    x, r = (torch.randn(9001, C, generator=g, device="cuda").to(dtype) for _ in range(2))
    group = 32 if C % 32 == 0 else None
    want = [*rms_norm(x, residual=r), *rms_norm_quantized(x, residual=r, group_size=group), *rms_norm_quantized(x)]
    large = torch.zeros(9001, dtype=torch.bool, device="cuda")
    large[[0, 7, 600, 4736, 4737, 8999]] = True
    x2, r2 = x.clone(), r.clone()
    x2[large] = (x[large].float() * 1e37).to(dtype)
    got = [*rms_norm(x2, residual=r2), *rms_norm_quantized(x2, residual=r2, group_size=group), *rms_norm_quantized(x2)]
    for a, b in zip(got, want):
        assert torch.equal(a[~large].float(), b[~large].float())
    y, _, _ = O.rms_norm(got[1][large], None, 1e-6)
    _close(got[0][large], y, y.abs(), "y")
    for codes, scales, h in ((got[2], got[3], got[1]), (got[5], got[6], x2)):
        y, _, _ = O.rms_norm(h[large], None, 1e-6)
        back = codes[large].double() * scales[large].double().repeat_interleave(C // scales.shape[1], -1)
        top = scales[large].double().repeat_interleave(C // scales.shape[1], -1) * 448
        assert float(((back - y).abs() - 2.0 ** -4 * y.abs() - 2.0 ** -10 / 448 * top - F * top).max()) <= 0


@pytest.mark.parametrize("group,C", [(32, 256), (64, 4096), (128, 8192), (32, 40064), (None, 256), (None, 1001), (None, 20000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_eight_bits_of_rows_with_an_infinity_or_a_nan(group, C, dtype):
    """As documented: codes and scale of an infinity's group are NaN, the others of its row zeros under the least scale; a NaN spoils its row."""
    from nitrix_b200.nn import rms_norm_quantized

    x = torch.randn(5, C, device="cuda").to(dtype)
    want = rms_norm_quantized(x, group_size=group)
    x[1, C // 2 + 3], x[3, 1] = -float("inf"), float("nan")
    codes, scales = rms_norm_quantized(x, group_size=group)
    size = group or C
    spoiled = torch.zeros(5, C // size, dtype=torch.bool, device="cuda")
    spoiled[1, (C // 2 + 3) // size] = True
    spoiled[3] = True
    assert torch.equal(scales.isnan(), spoiled) and torch.equal(codes.float().isnan(), spoiled.repeat_interleave(size, 1))
    rest = ~spoiled[1]
    assert not bool(codes[1].float()[rest.repeat_interleave(size)].any()) and bool((scales[1][rest] == 2.0 ** -100 * torch.tensor(1 / 448, device="cuda")).all())
    for row in (0, 2, 4):
        assert torch.equal(codes[row].float(), want[0][row].float()) and torch.equal(scales[row], want[1][row])
