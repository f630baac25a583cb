"""The operators of a decoder's attention layer, as far as they go without a GPU: refusals at the C entries, what the oracles
compute, the frequencies."""
import ctypes as C
import math
import random

import pytest
import torch

from oracle import decoder_oracle as O


def test_the_entry_points_refuse_what_is_no_parameter_block():
    from nitrix_b200 import _cabi

    lib = _cabi.lib()
    block = (C.c_char * 1024)()
    out, kernel = C.c_size_t(0), C.c_int(0)
    for name in ("nb200_rotary", "nb200_cache_append", "nb200_cache_fork", "nb200_cache_compact", "nb200_decode", "nb200_packed_fwd",
                 "nb200_packed_bwd"):
        for p in (None, block):      # (a struct_size of zero is nobody's)
            assert getattr(lib, name)(p, None) == _cabi.ERR_INVALID, name
            assert "struct_size" in _cabi.last_error()
    for name in ("nb200_cache_workspace_bytes", "nb200_decode_workspace_bytes"):
        assert getattr(lib, name)(block, C.byref(out)) == _cabi.ERR_INVALID, name
    assert lib.nb200_packed_workspace_bytes(block, 0, C.byref(out)) == _cabi.ERR_INVALID
    assert lib.nb200_packed_plan(block, 0, C.byref(kernel)) == _cabi.ERR_INVALID


@pytest.mark.skipif(torch.cuda.is_available(), reason="there is a GPU")
def test_there_is_no_host_path():
    from nitrix_b200 import NitrixBackendError
    from nitrix_b200.nn import packed_attention, rotary_embedding, rotary_frequencies

    q = torch.zeros(4, 2, 64)
    with pytest.raises(NitrixBackendError):
        rotary_embedding(q, None, torch.arange(4).int(), rotary_frequencies((32,)))
    with pytest.raises(NitrixBackendError):
        packed_attention(q, q, q, torch.tensor([0, 4]).int())


def test_frequencies():
    from nitrix_b200.nn import rotary_frequencies

    f = rotary_frequencies((3, 2), base=100.0)
    assert f.dtype == torch.float32
    assert torch.allclose(f, torch.tensor([1.0, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3), 1.0, 0.1]), rtol=1e-6)
    for sections, base in (((), 10.0), ((-1,), 10.0), ((4,), 0.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(sections, base=base)


@pytest.mark.parametrize("causal", [False, True])
def test_the_packed_oracle_against_differentiation(causal):
    g = torch.Generator().manual_seed(1)
    lq, lk = [5, 0, 9, 1], [7, 3, 4, 1]
    q, dout = (torch.randn(15, 4, 8, generator=g, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(15, 2, 8, generator=g, dtype=torch.float64) for _ in range(2))
    for t in (q, k, v):
        t.requires_grad_(True)
    out, sq, sk = [], 0, 0
    for a, b in zip(lq, lk):
        kk, vv = (t[sk:sk + b].repeat_interleave(2, dim=1) for t in (k, v))
        s = torch.einsum("ihd,jhd->hij", q[sq:sq + a], kk) * 0.7
        seen = torch.ones(a, b, dtype=torch.bool)
        if causal:
            seen = torch.arange(b)[None] <= torch.arange(a)[:, None] + b - a
        p = torch.where(seen, torch.exp(s), torch.zeros(()).double())
        out.append(torch.einsum("hij,jhd->ihd", p / p.sum(-1, keepdim=True).clamp(min=1e-300), vv))
        sq, sk = sq + a, sk + b
    out = torch.cat(out)
    grads = torch.autograd.grad(out, [q, k, v], dout)
    want = O.packed(q.detach(), k.detach(), v.detach(), lq, lk, 0.7, causal, dout)
    for name, value in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)):
        assert float((want[name][0] - value).abs().max()) < 1e-12, name
        assert bool((want[name][1] >= want[name][0].abs() - 1e-12).all())


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_rotary_oracle_turns_pairs(interleaved):
    x = torch.randn(3, 2, 10, dtype=torch.float64)
    pos, freq = torch.tensor([[0.0], [1.0], [2.5]]), torch.tensor([0.5, 1.5])
    y = O.rotary(x, pos, freq, (2,), interleaved)
    for n in range(3):
        for j in range(2):
            a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + 2)
            angle = float(pos[n, 0]) * float(freq[j])
            z = complex(float(x[n, 1, a]), float(x[n, 1, b])) * complex(math.cos(angle), math.sin(angle))
            assert abs(complex(float(y[n, 1, a]), float(y[n, 1, b])) - z) < 1e-12
    assert torch.equal(y[..., 4:], x[..., 4:])
    assert float((O.rotary(y, pos, freq, (2,), interleaved, inverse=True) - x).abs().max()) < 1e-12


def test_the_cache_model_keeps_every_token():
    rng = random.Random(0)
    m = O.CacheModel(60, 4, 5, 10)
    told, fresh = [[] for _ in range(5)], 0
    for _ in range(200):
        n = len(m.lengths)
        what = rng.choice(["append", "append", "fork", "compact"])
        if what == "append":
            new = [list(range(fresh + 3 * i, fresh + 3 * i + rng.randint(0, 3))) for i in range(n)]
            fresh += 3 * n
            m.append(new)
            told = [(old + tokens)[:m.lengths[i]] for i, (old, tokens) in enumerate(zip(told, new))]
        elif what == "fork":
            parents = [rng.randint(-1, n - 1) for _ in range(5)]
            m.fork(parents)
            told = [told[p][:m.lengths[i]] if p >= 0 else [] for i, p in enumerate(parents)]
        else:
            m.compact()
            live = {p for row in m.table for p in row}
            assert live == set(range(len(live)))
        assert [m.tokens(i) for i in range(len(m.lengths))] == told
        reached = [p for row in m.table for p in row]
        assert not set(reached) & set(m.free) and len(set(reached)) + len(m.free) == 60
