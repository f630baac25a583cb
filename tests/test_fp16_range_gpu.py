"""Dense fp16 attention whose row statistics leave the range of fp16."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _plain(q, k, v, dout, scale, mask=None):
    q, k, v = (t.double().requires_grad_(True) for t in (q, k, v))
    s = scale * q @ k.transpose(-1, -2)
    if mask is not None:
        s = s.masked_fill(~mask, float("-inf"))
    p = torch.softmax(s, -1)
    out = p @ v
    return [p.detach(), out.detach(), *torch.autograd.grad(out, (q, k, v), dout.double())]


def _grads(q, k, v, dout, **kw):
    from nitrix_b200.nn import scaled_dot_product_attention

    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = scaled_dot_product_attention(*leaves, **kw)
    return [out.detach(), *torch.autograd.grad(out, leaves, dout)]


def _inputs(D, S=200):
    g = torch.Generator(device="cuda").manual_seed(D)
    return [torch.randn(2, 3, S, D, generator=g, device="cuda").half() for _ in range(4)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("masked", [False, True])
def test_products_with_the_cotangent_of_millions(D, masked):
    """v = 200 and dout = 1000: delta is 1.3e7 at head dim 64 and 2.6e7 at 128.  dS, and with it dq and dk, is zero; delta comes from
    an output that is good to 2^-10, and so is P."""
    q, k, v, dout = _inputs(D)
    v, dout = v * 0 + 200, dout * 0 + 1000
    mask = torch.rand(2, 1, 200, 200, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) > 0.3 if masked else None
    if masked:
        mask[..., 0] = True
    p, out, dq, dk, dv = _plain(q, k, v, dout, D ** -0.5, mask)
    got = _grads(q, k, v, dout, mask=mask)
    noise = 2.0 ** -10 * D * 2e5 * D ** -0.5
    bounds = (2 * 2.0 ** -10 * 200 + 0 * out, noise * p @ k.double().abs() + 1e-3, noise * p.transpose(-1, -2) @ q.double().abs() + 1e-3,
              2 * 2.0 ** -10 * p.sum(-2)[..., None] * 1000 + 0 * dv)
    for name, a, b, bound in zip(("out", "dq", "dk", "dv"), got, (out, dq, dk, dv), bounds):
        assert float(((a.double() - b).abs() - bound).max()) <= 0, name


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scale", [1e-5, 1e-7, 1e-9, 1e-12])
def test_scales_far_below_one(D, scale):
    """Probabilities are equal to within 1e-3: out and dv are means and sums, of which fp16 keeps 2^-10; dq and dk are below fp16."""
    q, k, v, dout = _inputs(D)
    p, out, dq, dk, dv = _plain(q, k, v, dout, scale)
    got = _grads(q, k, v, dout, scale=scale)
    bounds = (2 * 2.0 ** -10 * p @ v.double().abs(), 1e-6 + 2.0 ** -8 * dq.abs(), 1e-6 + 2.0 ** -8 * dk.abs(),
              2 * 2.0 ** -10 * p.transpose(-1, -2) @ dout.double().abs())
    for name, a, b, bound in zip(("out", "dq", "dk", "dv"), got, (out, dq, dk, dv), bounds):
        assert float(((a.double() - b).abs() - bound).max()) <= 1e-6, name


@pytest.mark.parametrize("D", [64, 128])
def test_equal_scores_of_millions(D):
    """Scores of 2e7 before the scale: lse is good to two roundings of 1/8, a factor of 2^(1/4) in the probabilities at most."""
    q, k, v, dout = _inputs(D)
    q, k = q * 0 + 400, k * 0 + 400
    p, out, dq, dk, dv = _plain(q, k, v, dout, D ** -0.5)
    got = _grads(q, k, v, dout)
    dp = dout.double() @ v.double().transpose(-1, -2)
    ds = p * (dp.abs() + (p * dp.abs()).sum(-1, keepdim=True)) * D ** -0.5
    bounds = (2 * 2.0 ** -10 * p @ v.double().abs(), 0.2 * ds @ k.double(), 0.2 * ds.transpose(-1, -2) @ q.double(),
              0.2 * p.transpose(-1, -2) @ dout.double().abs())
    for name, a, b, bound in zip(("out", "dq", "dk", "dv"), got, (out, dq, dk, dv), bounds):
        assert float(((a.double() - b).abs() - bound).max()) <= 1e-3, name
