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
