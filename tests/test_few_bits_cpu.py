"""The norm and the cache in few bits, as far as they go without a GPU: refusals, and what the oracles compute."""
import ctypes as C

import pytest
import torch

from oracle import few_bits_oracle as O


def test_the_entry_points_refuse_what_is_no_parameter_block():
    from nitrix_b200 import _cabi

    lib = _cabi.lib()
    block = (C.c_char * 1024)()
    out = C.c_size_t(0)
    for name in ("nb200_rms_norm_fwd", "nb200_rms_norm_bwd", "nb200_cache_append_quantized", "nb200_cache_fork_quantized",
                 "nb200_cache_compact_quantized", "nb200_cache_read", "nb200_decode_quantized"):
        for p in (None, block):      # (a struct_size of zero is nobody's)
            assert getattr(lib, name)(p, None) == _cabi.ERR_INVALID, name
            assert "struct_size" in _cabi.last_error()
    for name in ("nb200_rms_norm_workspace_bytes", "nb200_decode_quantized_workspace_bytes"):
        assert getattr(lib, name)(block, C.byref(out)) == _cabi.ERR_INVALID, name
        assert getattr(lib, name)(block, None) == _cabi.ERR_INVALID, name


class _Rms(C.Structure):
    _fields_ = [("struct_size", C.c_size_t)] + [(n, C.c_void_p) for n in ("x", "residual", "weight", "y", "sum", "rstd", "scales", "dy", "dsum", "dx", "dweight", "workspace")] + \
        [("workspace_bytes", C.c_size_t), ("rows", C.c_int64), ("channels", C.c_int32), ("dtype", C.c_int32), ("weight_dtype", C.c_int32), ("group", C.c_int32),
         ("eps", C.c_float), ("reserved", C.c_int32)]


def _rms(**kw):
    p = _Rms(struct_size=C.sizeof(_Rms), rows=3, channels=64, dtype=1, weight_dtype=1, eps=1e-6, x=256, y=256, dy=256, dx=256, rstd=256)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change", [dict(dtype=7), dict(weight_dtype=2), dict(rows=-1), dict(channels=0), dict(channels=(1 << 30) + 1), dict(rows=1 << 32), dict(x=None), dict(y=None),
                                    dict(residual=256), dict(scales=256, group=48), dict(scales=256, group=128), dict(scales=256, group=32, x=264)])
def test_the_norm_refuses(change):
    from nitrix_b200 import _cabi

    assert _cabi.lib().nb200_rms_norm_fwd(C.byref(_rms(**change)), None) < 0
    assert _cabi.last_error().startswith("rms_norm_fwd")


@pytest.mark.parametrize("change", [dict(dy=None), dict(dx=None), dict(rstd=None), dict(weight_dtype=2)])
def test_the_norm_s_gradient_refuses(change):
    from nitrix_b200 import _cabi

    assert _cabi.lib().nb200_rms_norm_bwd(C.byref(_rms(**change)), None) < 0
    assert _cabi.last_error().startswith("rms_norm_bwd")


class _Pages(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_stride", C.c_int64 * 3), ("v_stride", C.c_int64 * 3)] + \
        [(n, C.c_int32) for n in ("pages", "heads", "page_size", "head_dim", "dtype", "reserved")]


class _Cache(C.Structure):
    _fields_ = [("struct_size", C.c_size_t), ("pages", _Pages)] + [(n, C.c_void_p) for n in ("table", "lengths", "free_pages", "free_range")] + \
        [("rows", C.c_int32), ("width", C.c_int32)] + \
        [(n, C.c_void_p) for n in ("new_table", "new_lengths", "new_free_pages", "new_free_range", "shortfall", "new_k", "new_v")] + \
        [("new_k_stride", C.c_int64 * 2), ("new_v_stride", C.c_int64 * 2), ("offsets", C.c_void_p), ("tokens", C.c_int64), ("parents", C.c_void_p),
         ("finished", C.c_void_p), ("new_rows", C.c_int32), ("reserved", C.c_int32), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class _Steps(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_stride", C.c_int64 * 3), ("v_stride", C.c_int64 * 3), ("bits", C.c_int32), ("reserved", C.c_int32)]


class _Quantized(C.Structure):
    _fields_ = [("struct_size", C.c_size_t), ("cache", _Cache), ("steps", _Steps)]


@pytest.mark.parametrize("change,code", [
    (dict(bits=5), "INVALID"), (dict(rows=0), "INVALID"), (dict(tokens=-1), "INVALID"), (dict(tokens=1 << 31), "INVALID"), (dict(offsets=None), "INVALID"),
    (dict(steps=None), "INVALID"), (dict(head_dim=80), "UNSUPPORTED"), (dict(heads=1 << 25), "UNSUPPORTED"), (dict(codes=264), "ALIGNMENT"), (dict(steps=260), "ALIGNMENT"), (dict(new_k=264), "ALIGNMENT"),
    (dict(token_stride=12), "ALIGNMENT"), (dict(slot_stride=40), "ALIGNMENT"), (dict(step_stride=3), "ALIGNMENT"),
    (dict(token_stride=1 << 34), "UNSUPPORTED"), (dict(slot_stride=1 << 35), "UNSUPPORTED"), (dict(step_stride=1 << 32), "UNSUPPORTED")])
def test_appending_refuses(change, code):
    from nitrix_b200 import _cabi

    c = {**dict(bits=4, heads=2, rows=1, tokens=2, offsets=256, steps=256, head_dim=64, codes=256, new_k=256, token_stride=128, slot_stride=32, step_stride=2), **change}
    pages = _Pages(k=c["codes"], v=256, k_stride=(512, 256, c["slot_stride"]), v_stride=(512, 256, 32), pages=4, heads=c["heads"], page_size=8, head_dim=c["head_dim"], dtype=1)
    cache = _Cache(struct_size=C.sizeof(_Cache), pages=pages, rows=c["rows"], width=3, new_k_stride=(c["token_stride"], 64), new_v_stride=(128, 64), tokens=c["tokens"],
                   offsets=c["offsets"], new_k=c["new_k"], new_v=256,
                   **{n: 256 for n in ("table", "lengths", "free_pages", "free_range", "new_lengths", "new_free_range", "shortfall")})
    steps = _Steps(k=c["steps"], v=256, k_stride=(32, 16, c["step_stride"]), v_stride=(32, 16, 2), bits=c["bits"])
    p = _Quantized(struct_size=C.sizeof(_Quantized), cache=cache, steps=steps)
    assert _cabi.lib().nb200_cache_append_quantized(C.byref(p), None) == getattr(_cabi, "ERR_" + code), _cabi.last_error()
    assert "cache_append_quantized" in _cabi.last_error()


class _Read(C.Structure):
    _fields_ = [("struct_size", C.c_size_t), ("pages", _Pages), ("steps", _Steps), ("table", C.c_void_p), ("lengths", C.c_void_p), ("rows", C.c_int32),
                ("width", C.c_int32)] + [(n, C.c_void_p) for n in ("offsets", "starts", "out_k", "out_v")] + [("tokens", C.c_int64)]


@pytest.mark.parametrize("change,code", [
    (dict(bits=3), "INVALID"), (dict(dtype=7), "INVALID"), (dict(tokens=1 << 31), "INVALID"), (dict(offsets=None), "INVALID"), (dict(out_v=None), "INVALID"),
    (dict(head_dim=48), "UNSUPPORTED"), (dict(codes=264), "ALIGNMENT"), (dict(out_v=264), "ALIGNMENT"), (dict(dtype=0, out_v=272), "ALIGNMENT"),
    (dict(heads=1 << 30), "UNSUPPORTED")])
def test_reading_refuses(change, code):
    from nitrix_b200 import _cabi

    c = {**dict(bits=4, dtype=1, tokens=2, offsets=256, head_dim=64, heads=2, codes=256, out_v=256), **change}
    pages = _Pages(k=c["codes"], v=256, k_stride=(512, 256, 32), v_stride=(512, 256, 32), pages=4, heads=c["heads"], page_size=8, head_dim=c["head_dim"], dtype=c["dtype"])
    steps = _Steps(k=256, v=256, k_stride=(32, 16, 2), v_stride=(32, 16, 2), bits=c["bits"])
    p = _Read(struct_size=C.sizeof(_Read), pages=pages, steps=steps, table=256, lengths=256, rows=1, width=3, offsets=c["offsets"], out_k=256, out_v=c["out_v"],
              tokens=c["tokens"])
    assert _cabi.lib().nb200_cache_read(C.byref(p), None) == getattr(_cabi, "ERR_" + code), _cabi.last_error()
    assert "cache_read" in _cabi.last_error()


class _Decode(C.Structure):
    _fields_ = [("struct_size", C.c_size_t), ("pages", _Pages), ("table", C.c_void_p), ("lengths", C.c_void_p), ("rows", C.c_int32), ("width", C.c_int32),
                ("q", C.c_void_p), ("out", C.c_void_p), ("q_stride", C.c_int64 * 2), ("q_heads", C.c_int32), ("scale", C.c_float), ("workspace", C.c_void_p),
                ("workspace_bytes", C.c_size_t)]


class _QuantizedDecode(C.Structure):
    _fields_ = [("struct_size", C.c_size_t), ("decode", _Decode), ("steps", _Steps)]


@pytest.mark.parametrize("change,code", [
    (dict(bits=2), "INVALID"), (dict(dtype=7), "INVALID"), (dict(heads=0), "INVALID"), (dict(page_size=0), "INVALID"), (dict(rows=-1), "INVALID"), (dict(q_heads=3), "INVALID"),
    (dict(q_heads=0), "INVALID"), (dict(q=None), "INVALID"), (dict(out=None), "INVALID"), (dict(table=None), "INVALID"), (dict(lengths=None), "INVALID"), (dict(codes=None), "INVALID"),
    (dict(steps=None), "INVALID"), (dict(head_dim=72), "UNSUPPORTED"), (dict(head_dim=288), "UNSUPPORTED"), (dict(rows=65536), "UNSUPPORTED"), (dict(codes=264), "ALIGNMENT"),
    (dict(slot_stride=40), "ALIGNMENT"), (dict(steps=260), "ALIGNMENT"), (dict(step_stride=3), "ALIGNMENT"), (dict(slot_stride=1 << 35), "UNSUPPORTED"),
    (dict(step_stride=1 << 32), "UNSUPPORTED"), (dict(workspace=None), "WORKSPACE"), (dict(short=1), "WORKSPACE"), (dict(workspace=264), "ALIGNMENT"), (dict(inner_size=8), "INVALID")])
def test_attention_over_codes_refuses(change, code):
    from nitrix_b200 import _cabi

    c = {**dict(bits=4, dtype=1, heads=2, page_size=8, rows=1, q_heads=4, q=256, out=256, table=256, lengths=256, codes=256, steps=256, head_dim=64, slot_stride=32, step_stride=2,
                workspace=256, short=0, inner_size=C.sizeof(_Decode)), **change}
    pages = _Pages(k=c["codes"], v=256, k_stride=(512, 256, c["slot_stride"]), v_stride=(512, 256, 32), pages=4, heads=c["heads"], page_size=c["page_size"], head_dim=c["head_dim"],
                   dtype=c["dtype"])
    steps = _Steps(k=c["steps"], v=256, k_stride=(32, 16, c["step_stride"]), v_stride=(32, 16, 2), bits=c["bits"])
    decode = _Decode(struct_size=c["inner_size"], pages=pages, table=c["table"], lengths=c["lengths"], rows=c["rows"], width=3, q=c["q"], out=c["out"], q_stride=(256, 64),
                     q_heads=c["q_heads"], scale=0.1, workspace=c["workspace"])
    p = _QuantizedDecode(struct_size=C.sizeof(_QuantizedDecode), decode=decode, steps=steps)
    need = C.c_size_t(0)
    if _cabi.lib().nb200_decode_quantized_workspace_bytes(C.byref(p), C.byref(need)) == 0:      # (what it says of the sizes alone is asked first)
        assert need.value > 0
    p.decode.workspace_bytes = need.value - c["short"]
    assert _cabi.lib().nb200_decode_quantized(C.byref(p), None) == getattr(_cabi, "ERR_" + code), _cabi.last_error()
    assert "decode_quantized" in _cabi.last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="there is a GPU")
def test_there_is_no_host_path():
    from nitrix_b200 import NitrixBackendError
    from nitrix_b200.nn import cache_read, quantized_cache, rms_norm, rms_norm_quantized

    x = torch.zeros(4, 64)
    cache = quantized_cache(4, 8, 1, 64, sequences=2, max_length=16, device="cpu")
    for call in (lambda: rms_norm(x), lambda: rms_norm_quantized(x), lambda: cache_read(cache, torch.zeros(3).int(), 0)):
        with pytest.raises(NitrixBackendError):
            call()


def test_caches_that_cannot_be():
    from nitrix_b200.nn import quantized_cache

    good = dict(pages=4, page_size=8, kv_heads=1, head_dim=64, bits=4, sequences=2, max_length=16, device="cpu")
    c = quantized_cache(**good)
    assert c.k_codes.shape == (4, 1, 8, 32) and c.k_steps.shape == (4, 1, 8, 2) and c.table.shape == (2, 2)
    assert quantized_cache(**{**good, "bits": 8}).v_codes.shape == (4, 1, 8, 64)
    for change in (dict(pages=0), dict(page_size=0), dict(kv_heads=0), dict(head_dim=0), dict(max_length=0), dict(bits=5), dict(head_dim=48)):
        with pytest.raises(ValueError):
            quantized_cache(**{**good, **change})


@pytest.mark.parametrize("weight", [False, True])
def test_the_norm_s_oracle_against_differentiation(weight):
    g = torch.Generator().manual_seed(3)
    h, dy, dsum = (torch.randn(6, 10, generator=g, dtype=torch.float64) for _ in range(3))
    w = torch.randn(10, generator=g, dtype=torch.float64).requires_grad_(True) if weight else None
    h.requires_grad_(True)
    y = h / torch.sqrt((h ** 2).sum(1, keepdim=True) / 10 + 0.01) * (1 if w is None else w)
    grads = torch.autograd.grad([y, h * 1], [h] if w is None else [h, w], [dy, dsum])
    got = O.rms_norm(h.detach(), None if w is None else w.detach(), 0.01)[0]
    dx, bound, dw, dw_bound = O.rms_norm_grads(h.detach(), None if w is None else w.detach(), 0.01, dy, dsum)
    assert float((got - y).abs().max()) < 1e-12 and float((dx - grads[0]).abs().max()) < 1e-12
    assert bool((bound >= dx.abs() - 1e-12).all()) and bool((dw_bound >= dw.abs() - 1e-12).all())
    if weight:
        assert float((dw - grads[1]).abs().max()) < 1e-12


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("D", [32, 96, 128])
def test_the_cache_s_oracle(bits, D):
    """Codes come back from their bytes, and a value is within half a step of its code's, one and a half at the far end."""
    g = torch.Generator().manual_seed(bits + D)
    x = torch.randn(50, 3, D, generator=g)
    x[0, 0] = 0
    x[1, 0, :32] = 7.0          # (all alike)
    codes, steps = O.quantize(x, bits)
    half = 1 << (bits - 1)
    assert int(codes.min()) >= 0 and int(codes.max()) <= 2 * half - 1
    rows = O.packed_codes(codes, bits)
    assert rows.shape[-1] == D * bits // 8
    back = O.values(rows, steps, bits)
    each = steps.double().repeat_interleave(32, -1)
    assert torch.equal(back, (codes - half).double() * each)
    err = (back - x.double()).abs()
    # a step is rounded to fp16, which the far end, half of them, feels most
    assert bool((err <= each.abs() * (0.5 + half * 2.0 ** -11) + each.abs() * (codes == 2 * half - 1)).all())
    assert torch.equal(back[0, 0], torch.zeros(D).double()) and torch.equal(back[1, 0, :32], torch.full((32,), 7.0).double())
    top = x.abs().unflatten(-1, (-1, 32)).amax(-1)
    assert bool((steps.double().abs() * half - top.double()).abs().le(top.double() * 2.0 ** -11).all())


def test_the_cache_s_oracle_at_the_ends_of_the_range():
    x = torch.zeros(5, 32)
    x[0, 3] = 3e38
    x[1, 3] = 1e-9
    x[2, 3], x[3, 4] = float("inf"), float("nan")
    x[4, 0], x[4, 1] = -1.0, 1.0
    codes, steps = O.quantize(x, 4)
    assert float(steps[0, 0]) == -65504.0 and float(steps[1, 0]) == 0.0 and bool(steps[2:4].isnan().all())
    assert codes[0].tolist() == [8, 8, 8, 0] + [8] * 28 and codes[1:4].unique().tolist() == [8]
    assert codes[4, :3].tolist() == [15, 0, 8]      # (of two of one size, the positive one has the code 0)
