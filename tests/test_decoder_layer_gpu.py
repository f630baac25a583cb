"""The example's layer: what it serves token by token is what its packed form computes for the whole sequences."""
import importlib.util
import pathlib

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = pathlib.Path(__file__).resolve().parent.parent


def _example():
    spec = importlib.util.spec_from_file_location("decoder_layer", ROOT / "examples" / "decoder_layer.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_served_tokens_are_those_of_the_whole_sequences():
    """Both forms round queries, keys, values, attention and output to bf16 at the same places; the attention's own error is half
    an ulp of sums of size one, the output's a further half ulp: 2^-6 of the largest output covers both forms' sums."""
    ex = _example()
    layer = ex.AttentionLayer()
    g = torch.Generator(device="cuda").manual_seed(3)
    prompts = [torch.randn(n, 256, generator=g, device="cuda").bfloat16() for n in (40, 7, 100, 16)]
    outputs, fed, compacted, cache = ex.serve(layer, prompts, beams=2, steps=8)
    parents = [i for i in range(4) for _ in range(2)]
    assert cache.lengths.tolist() == [prompts[p].shape[0] + 8 for p in parents]
    whole = [torch.cat([prompts[p], *[t[i:i + 1] for t in fed]]) for i, p in enumerate(parents)]
    offsets, positions = ex.pack([w.shape[0] for w in whole])
    with torch.no_grad():
        want = layer.packed(torch.cat(whole), positions, offsets)
    for i, p in enumerate(parents):
        rows = want[int(offsets[i]) + prompts[p].shape[0] - 1:int(offsets[i + 1])]
        got = torch.stack([o[i] for o in outputs])
        assert float((got.float() - rows.float()).abs().max()) <= 2.0 ** -6 * float(want.float().abs().max())
    kept = [0 if i % 3 == 2 else n for i, n in enumerate(cache.lengths.tolist())]
    assert compacted.lengths.tolist() == kept
    pages = {x for row, n in zip(compacted.table.tolist(), kept) for x in row[:-(-n // 16)]}
    assert pages == set(range(len(pages)))
    assert compacted.free_range.tolist() == [0, 256 - len(pages)]


def test_training_lowers_the_loss():
    ex = _example()
    losses = ex.train(ex.AttentionLayer(), [120, 3, 300, 1, 77], steps=12)
    assert losses[-1] < 0.7 * losses[0]
