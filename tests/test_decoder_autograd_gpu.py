"""The differentiable operators of a decoder layer: what autograd asks of them, and what they refuse."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rotary():
    from nitrix_b200.nn import rotary_embedding, rotary_frequencies

    g = torch.Generator(device="cuda").manual_seed(1)
    leaves = [torch.randn(50, h, 64, generator=g, device="cuda").requires_grad_(True) for h in (4, 2)]
    freq, pos = rotary_frequencies((32,), device="cuda"), torch.arange(50, device="cuda").int()
    return leaves, lambda q, k: torch.cat(rotary_embedding(q, k, pos, freq), dim=1)


def _packed(dtype):
    from nitrix_b200.nn import packed_attention

    g = torch.Generator(device="cuda").manual_seed(2)
    leaves = [torch.randn(430, h, 64, generator=g, device="cuda").to(dtype).requires_grad_(True) for h in (4, 2, 2)]
    offsets = torch.tensor([0, 130, 130, 430], dtype=torch.int32, device="cuda")
    return leaves, lambda q, k, v: packed_attention(q, k, v, offsets)


_OPS = {"rotary": _rotary, "packed bf16": lambda: _packed(torch.bfloat16), "packed f16": lambda: _packed(torch.float16),
        "packed f32": lambda: _packed(torch.float32)}


@pytest.mark.parametrize("op", _OPS)
def test_gradients_of_some_operands_and_on_another_stream_and_through_hooks(op):
    leaves, fn = _OPS[op]()
    want = torch.autograd.grad(fn(*leaves).float().square().sum(), leaves)

    def close(a, b):   # (sums added in any order)
        assert float((a.float() - b.float()).norm()) <= 1e-2 * float(b.float().norm())

    for i, leaf in enumerate(leaves):
        only = [t if j == i else t.detach() for j, t in enumerate(leaves)]
        close(torch.autograd.grad(fn(*only).float().square().sum(), [leaf])[0], want[i])
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (saved.append(1), t.cpu())[1], lambda t: t.cuda()):
        y = fn(*leaves)
    assert saved
    for a, b in zip(torch.autograd.grad(y.float().square().sum(), leaves), want):
        close(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.autograd.grad(fn(*leaves).float().square().sum(), leaves)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        close(a, b)
    with torch.no_grad():
        assert not fn(*leaves).requires_grad


@pytest.mark.parametrize("op", _OPS)
def test_what_has_no_rule_is_refused(op):
    leaves, fn = _OPS[op]()
    rest = [t.detach() for t in leaves[1:]]
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: fn(x, *rest))(torch.stack([leaves[0].detach()] * 2))
    x = leaves[0]
    (gx,) = torch.autograd.grad(fn(x, *rest).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.float().sum(), x)
    if op != "rotary":      # (its gradient needs neither operand)
        z = leaves[0] * 1
        y = fn(z, *rest)
        z.add_(1)
        with pytest.raises(RuntimeError, match="inplace"):
            y.float().sum().backward()


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("op", _OPS)
def test_forward_mode_is_not_implemented(op, grad):
    # (without gradients as well: a result without a tangent would be taken for one that does not depend on the operand)
    leaves, fn = _OPS[op]()
    leaves = [t.detach().requires_grad_(grad) for t in leaves]
    for i in range(len(leaves)):
        with pytest.raises(NotImplementedError), torch.autograd.forward_ad.dual_level():
            fn(*(torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(leaves)))


def test_forward_mode_through_a_cache_is_not_implemented():
    from nitrix_b200.nn import cache_append, decode_attention, paged_cache

    dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
    cache = paged_cache(8, 4, 2, 64, sequences=3, max_length=16)
    k = torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    q = torch.zeros(3, 4, 64, device="cuda", dtype=torch.bfloat16)
    offsets = torch.arange(4, device="cuda").int()
    for call in (lambda: decode_attention(dual(q), cache), lambda: decode_attention(q, cache._replace(k_pages=dual(cache.k_pages))),
                 lambda: decode_attention(q, cache._replace(v_pages=dual(cache.v_pages))), lambda: cache_append(cache, dual(k), k, offsets),
                 lambda: cache_append(cache, k, dual(k), offsets), lambda: cache_append(cache._replace(v_pages=dual(cache.v_pages)), k, k, offsets)):
        with pytest.raises(NotImplementedError, match="forward-mode"), torch.autograd.forward_ad.dual_level():
            call()


def test_forward_mode_of_dense_attention_without_gradients_is_not_implemented():
    from nitrix_b200.nn import scaled_dot_product_attention

    x = torch.randn(1, 2, 40, 64, device="cuda").bfloat16()
    for i in range(3):
        with pytest.raises(NotImplementedError), torch.autograd.forward_ad.dual_level():
            scaled_dot_product_attention(*(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)) if i == j else x for j in range(3)))
