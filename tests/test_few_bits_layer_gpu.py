"""The operators in few bits as a decoder layer uses them together: norm, rotary positions, a cache in 4 or 8 bits that is written,
read back for the next chunk of a prompt, and attended to token by token."""
import importlib.util
import pathlib

import pytest
import torch

from oracle import decoder_oracle as D
from oracle import few_bits_oracle as O

pytestmark = pytest.mark.gpu

ROOT = pathlib.Path(__file__).resolve().parent.parent


def _example():
    spec = importlib.util.spec_from_file_location("decoder_layer", ROOT / "examples" / "decoder_layer.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _quantized(x, bits):
    codes, steps = O.quantize(x, bits)
    return O.values(O.packed_codes(codes, bits), steps, bits)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 64), (4, 4, 128)])
def test_prompts_in_chunks_and_then_token_by_token(bits, heads, kv_heads, head_dim):
    """Every step against attention in 64 bits over what the oracle says the cache holds.  Keys and values read back are rounded once
    to bf16, probabilities and results too (2^-8 each, of the sums of magnitudes); the output's product has its own half ulp."""
    from nitrix_b200.nn import quantized_cache, rms_norm

    ex = _example()
    layer = ex.AttentionLayer(width=128, heads=heads, kv_heads=kv_heads, head_dim=head_dim)
    g = torch.Generator(device="cuda").manual_seed(3)
    chunks = [[40, 7, 0, 100], [16, 1, 33, 60], [0, 80, 1, 5]]
    cache = quantized_cache(100, 16, kv_heads, head_dim, bits=bits, sequences=4, max_length=300)
    held = [[torch.zeros(0, kv_heads, head_dim, dtype=torch.float64, device="cuda")] * 2 for _ in range(4)]
    with torch.no_grad():
        for lengths in chunks:
            x = torch.randn(sum(lengths), 128, generator=g, device="cuda").bfloat16()
            offsets, _ = ex.pack(lengths)
            positions = torch.cat([torch.arange(h[0].shape[0], h[0].shape[0] + n) for h, n in zip(held, lengths)]).int().cuda()
            q, k, v = layer.project(x, positions)
            at = 0
            for i, n in enumerate(lengths):
                held[i] = [torch.cat([old, _quantized(new[at:at + n], bits)]) for old, new in zip(held[i], (k, v))]
                at += n
            out, cache = layer.chunk(x, positions, offsets, cache, 400)
            assert cache.lengths.tolist() == [h[0].shape[0] for h in held]
            keys, values = (torch.cat([h[j] for h in held]).bfloat16() for j in range(2))
            want = D.packed(q, keys, values, lengths, cache.lengths.tolist(), head_dim ** -0.5, True)["out"]
            o, bound = want[0].flatten(1), want[1].flatten(1)
            w = layer.w_out.double()
            err = (out.double() - o @ w.T).abs() - 2.0 ** -6 * (bound @ w.abs().T)
            assert float(err.max()) <= 1e-6, float(err.max())
        gain = (1 + 0.1 * torch.randn(128, generator=g, device="cuda")).bfloat16()
        stream = torch.randn(4, 128, generator=g, device="cuda").bfloat16()
        for _ in range(5):
            x = torch.randn(4, 128, generator=g, device="cuda").bfloat16()
            before = cache
            out, after, cache = layer.block(x, stream, gain, cache)
            assert torch.equal(after, O.stream_sum(x, stream))
            y, _ = rms_norm(x, gain, residual=stream)      # (the same numbers every time)
            exact, _, _ = O.rms_norm(after, gain, 1e-6)
            assert float(((y.double() - exact).abs() - 2.0 ** -8 * 1.01 * exact.abs()).max()) <= 0
            q, k, v = layer.project(y, before.lengths)
            held = [[torch.cat([old, _quantized(new[i:i + 1], bits)]) for old, new in zip(h, (k, v))] for i, h in enumerate(held)]
            keys, values = (torch.cat([h[j] for h in held]) for j in range(2))
            want = D.packed(q, keys, values, [1] * 4, cache.lengths.tolist(), head_dim ** -0.5, True)["out"]
            w = layer.w_out.double()
            err = (out.double() - want[0].flatten(1) @ w.T).abs() - 2.0 ** -6 * (want[1].flatten(1) @ w.abs().T)
            assert float(err.max()) <= 1e-6, float(err.max())
            stream = after


@pytest.mark.parametrize("bits", [4, 8])
def test_the_example_serves_from_few_bits(bits):
    """It runs, beams are forked and the pool is packed; how far its tokens are from the full cache's is the quantisation's affair."""
    ex = _example()
    layer = ex.AttentionLayer()
    prompts = [torch.randn(n, 256, generator=torch.Generator(device="cuda").manual_seed(n), device="cuda").bfloat16() for n in (40, 7, 100, 16)]
    outputs, fed, compacted, cache = ex.serve(layer, prompts, beams=2, steps=8, bits=bits)
    assert len(outputs) == 9 and all(bool(o.isfinite().all()) for o in outputs)
    assert cache.lengths.tolist() == [n + 8 for n in (40, 40, 7, 7, 100, 100, 16, 16)]
    kept = [0 if i % 3 == 2 else n for i, n in enumerate(cache.lengths.tolist())]
    assert compacted.lengths.tolist() == kept
    pages = {x for row, n in zip(compacted.table.tolist(), kept) for x in row[:-(-n // 16)]}
    assert pages == set(range(len(pages)))


def test_a_norm_is_trained_in_front_of_the_layer():
    """Gradients of the norm and of the sum beside it through what follows, against 64 bits."""
    from nitrix_b200.nn import rms_norm

    x, r = (torch.randn(60, 96, generator=torch.Generator(device="cuda").manual_seed(s), device="cuda").requires_grad_(True) for s in (1, 2))
    w = torch.ones(96, device="cuda", requires_grad=True)
    mix = torch.randn(96, 96, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda") / 10
    y, h = rms_norm(x, w, residual=r)
    loss = ((y @ mix).tanh() + h).square().mean()
    grads = torch.autograd.grad(loss, [x, r, w])
    ops = [t.detach().double().requires_grad_(True) for t in (x, r, w)]
    h64 = ops[0] + ops[1]
    y64, _, _ = O.rms_norm(h64, ops[2], 1e-6)
    want = torch.autograd.grad(((y64 @ mix.double()).tanh() + h64).square().mean(), ops)
    for a, b in zip(grads, want):
        # (a product of 96 terms and a few factors in fp32, TF32 off)
        assert float((a.double() - b).norm()) <= 1e-5 * float(b.norm())
