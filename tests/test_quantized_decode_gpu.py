"""Attention over a cache in 4 and 8 bits: head dims, queries and values that the other tests of it leave out.

The bounds are those of ``test_quantized_cache_gpu.py``: 2^-11 of the sums of magnitudes for 16-bit operands' probabilities on the tensor
cores, fp32's roundings of scores and sums, half an ulp of the result.
"""
import ctypes as C

import pytest
import torch

from oracle import few_bits_oracle as O

pytestmark = pytest.mark.gpu

HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _filled(lengths, page_size, Hk, dim, bits, seed=0, sign=None):
    """A cache of random codes and steps in pages of random order, NaN steps wherever no token is; ``sign``: keys of one sign."""
    from nitrix_b200.nn import quantized_cache

    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page_size) for n in lengths]
    pool = sum(need) + 3
    c = quantized_cache(pool, page_size, Hk, dim, bits=bits, sequences=len(lengths), max_length=max(1, *need) * page_size)
    for t in c[:2]:
        t.random_(0, 256)
    for t in c[2:4]:
        t.fill_(float("nan"))
    order, at = torch.randperm(pool, generator=g, device="cuda").int(), 0
    for i, n in enumerate(lengths):
        c.table[i, :need[i]] = order[at:at + need[i]]
        at += need[i]
        t = torch.arange(n, device="cuda")
        where = c.table[i].long()[t // page_size], slice(None), t % page_size
        for j, (codes, steps) in enumerate(((c.k_codes, c.k_steps), (c.v_codes, c.v_steps))):
            x = torch.randn(n, Hk, dim, generator=g, device="cuda")
            if sign is not None and j == 0:
                x = sign * x.abs()
            a, b = O.quantize(x, bits)
            codes[where], steps[where] = O.packed_codes(a, bits), b
    c.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    return c


def _bound(got, q, cache, lengths, bits, scale, p_rounding):
    k, v = O.cache_values(cache, bits)
    want, spread, reach = O.decode(q, k, v, cache.table, lengths, scale)
    bound = HALF[q.dtype] * want.abs() + (p_rounding + 2 * 16 * 2.0 ** -24 * (1 + reach) + 2.0 ** -20) * 2 * spread
    return want, (got.double() - want).abs() - bound - 2.0 ** -25


def _check(q, cache, lengths, bits, scale=None):
    from nitrix_b200.nn import decode_attention

    scale = q.shape[-1] ** -0.5 if scale is None else scale
    got = decode_attention(q, cache, scale=scale)
    assert got.dtype == q.dtype and got.shape == q.shape and bool(got.isfinite().all())
    _, err = _bound(got, q, cache, lengths, bits, scale, 0 if q.dtype == torch.float32 else 2.0 ** -11)
    assert float(err.max()) <= 0, float(err.max())
    return got


LENGTHS = [0, 1, 15, 16, 17, 63, 65, 129, 700]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [160, 192, 224])
@pytest.mark.parametrize("Hk,G", [(1, 1), (2, 3), (1, 9)])
def test_head_dims_between_128_and_256(bits, dtype, dim, Hk, G):
    cache = _filled(LENGTHS, 16, Hk, dim, bits, seed=dim + G)
    _check(torch.randn(len(LENGTHS), Hk * G, dim, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype), cache, LENGTHS, bits)


class _Pages(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_stride", C.c_int64 * 3), ("v_stride", C.c_int64 * 3)] + \
        [(n, C.c_int32) for n in ("pages", "heads", "page_size", "head_dim", "dtype", "reserved")]


class _Decode(C.Structure):
    _fields_ = [("struct_size", C.c_size_t), ("pages", _Pages), ("table", C.c_void_p), ("lengths", C.c_void_p), ("rows", C.c_int32), ("width", C.c_int32),
                ("q", C.c_void_p), ("out", C.c_void_p), ("q_stride", C.c_int64 * 2), ("q_heads", C.c_int32), ("scale", C.c_float), ("workspace", C.c_void_p),
                ("workspace_bytes", C.c_size_t)]


class _Steps(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_stride", C.c_int64 * 3), ("v_stride", C.c_int64 * 3), ("bits", C.c_int32), ("reserved", C.c_int32)]


class _QuantizedDecode(C.Structure):
    _fields_ = [("struct_size", C.c_size_t), ("decode", _Decode), ("steps", _Steps)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("Hk,G", [(2, 1), (1, 2), (2, 3), (1, 4), (2, 9)])
def test_16_bit_queries_off_a_16_byte_boundary(bits, dtype, dim, Hk, G):
    """Where the library is called as such (the Python entry point copies such queries first): the fp32 units take them, with fp32's error."""
    from nitrix_b200 import _cabi

    cache = _filled(LENGTHS, 16, Hk, dim, bits, seed=G)
    rows, H = len(LENGTHS), Hk * G
    flat = torch.randn(rows * H * dim + 1, device="cuda").to(dtype)
    q = flat[1:].view(rows, H, dim)
    assert q.data_ptr() % 16
    out = torch.full_like(q, float("nan"))
    pages = _Pages(k=cache.k_codes.data_ptr(), v=cache.v_codes.data_ptr(), k_stride=cache.k_codes.stride()[:3], v_stride=cache.v_codes.stride()[:3],
                   pages=cache.k_codes.shape[0], heads=Hk, page_size=16, head_dim=dim, dtype=_cabi.BF16 if dtype == torch.bfloat16 else _cabi.F16)
    steps = _Steps(k=cache.k_steps.data_ptr(), v=cache.v_steps.data_ptr(), k_stride=cache.k_steps.stride()[:3], v_stride=cache.v_steps.stride()[:3], bits=bits)
    decode = _Decode(struct_size=C.sizeof(_Decode), pages=pages, table=cache.table.data_ptr(), lengths=cache.lengths.data_ptr(), rows=rows, width=cache.table.shape[1],
                     q=q.data_ptr(), out=out.data_ptr(), q_stride=(H * dim, dim), q_heads=H, scale=dim ** -0.5)
    p = _QuantizedDecode(struct_size=C.sizeof(_QuantizedDecode), decode=decode, steps=steps)
    need = C.c_size_t(0)
    lib = _cabi.lib()
    assert lib.nb200_decode_quantized_workspace_bytes(C.byref(p), C.byref(need)) == 0, _cabi.last_error()
    workspace = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    p.decode.workspace, p.decode.workspace_bytes = workspace.data_ptr(), need.value
    assert lib.nb200_decode_quantized(C.byref(p), C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0, _cabi.last_error()
    _, err = _bound(out, q, cache, LENGTHS, bits, dim ** -0.5, 0)
    assert not bool(out.isnan().any()) and float(err.max()) <= 0, float(err.max())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 96])
def test_queries_and_keys_of_one_sign(bits, dtype, dim):
    """The middle of the codes' range comes off the sums of the codes, which are then all of one size; scores lie close together or far."""
    lengths = [300, 33, 1]
    g = torch.Generator(device="cuda").manual_seed(2)
    for sign in (1.0, -1.0):
        cache = _filled(lengths, 16, 2, dim, bits, seed=3, sign=sign)
        q = torch.randn(3, 8, dim, generator=g, device="cuda").abs().to(dtype)
        for scale in (None, 1.0):
            _check(q, cache, lengths, bits, scale)
            _check(torch.full_like(q, 1.5), cache, lengths, bits, scale)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
def test_groups_of_values_beyond_fp16_of_each_other(bits, dtype, dim):
    """16-bit queries: an element is off by 2^-11 of its terms and, per token, by 2^-32 of its head's largest product of a probability and a
    step times the half of the codes' range; fp32 queries have no such term."""
    from nitrix_b200.nn import decode_attention

    lengths = [900, 40]
    cache = _filled(lengths, 16, 2, dim, bits)
    size = torch.tensor([3e4, 1e-5, 1.0, 1e-7], device="cuda")[:dim // 32]
    cache.v_steps.copy_((cache.v_steps.float().sign() * size).half())
    q = torch.randn(2, 4, dim, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").to(dtype)
    scale, half = 0.3, 1 << (bits - 1)
    got = decode_attention(q, cache, scale=scale)
    k, _ = O.cache_values(cache, bits)
    want, err = _bound(got, q, cache, lengths, bits, scale, 2.0 ** -11)
    # (of values up to 2.4e5 fp16 cannot hold every mean: from 65520 on an infinity is the number next to it)
    beyond = (want.abs() >= 65520 * (1 - 2.0 ** -10)) & (got.double() == want.sign() * float("inf"))
    assert bool((dtype == torch.float16) | ~beyond.any())
    err[beyond] = 0
    largest = 0.0
    for i, n in enumerate(lengths):
        t = torch.arange(n, device="cuda")
        pages = cache.table[i].long()[t // 16]
        for h in range(4):
            p = torch.softmax(scale * k[pages, h // 2, t % 16] @ q[i, h].double(), 0)
            top = float((p * cache.v_steps[pages, h // 2, t % 16].double().abs().amax(-1)).max())
            largest = max(largest, float(err[i, h].max()) - n * 2.0 ** -32 * top * half)
    assert largest <= 0, largest
    _check(q.float(), cache, lengths, bits, scale)


def test_batched_tensors_are_refused():
    """The functions have no batching rule: ``vmap`` over them raises, and nothing is written."""
    from nitrix_b200.nn import cache_append, cache_read, decode_attention, rms_norm, rms_norm_quantized

    cache = _filled([20, 3], 16, 2, 64, 4)
    before = [t.clone() for t in cache]
    x, w = torch.randn(3, 5, 64, device="cuda"), torch.ones(64, device="cuda")
    k, offsets = torch.randn(3, 2, 2, 64, device="cuda"), torch.arange(3, device="cuda").int()
    q = torch.randn(3, 2, 4, 64, device="cuda")
    calls = [(lambda t: rms_norm(t, w), x), (lambda t: rms_norm(x[0], t), torch.ones(3, 64, device="cuda")), (lambda t: rms_norm(x[0], w, residual=t), x),
             (lambda t: rms_norm_quantized(t, w)[0].float(), x), (lambda t: rms_norm(t, w), x.clone().requires_grad_(True)), (lambda t: cache_append(cache, t, t, offsets).lengths, k),
             (lambda t: cache_read(cache, t, 2)[0], offsets.repeat(3, 1)), (lambda t: decode_attention(t, cache), q)]
    for call, batched in calls:
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(batched)
    for a, b in zip(cache, before):
        assert torch.equal(a.nan_to_num(), b.nan_to_num())
