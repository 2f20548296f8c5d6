"""The 8-bit operators' refusals, without a GPU."""
import ctypes

import pytest
import torch

from packkv_amd import _lib, ops

F8 = torch.float8_e4m3fn


def test_host_tensors_are_refused():
    x, w = torch.zeros(2, 128, dtype=torch.float16), torch.ones(128, dtype=torch.float16)
    e = {"codes": torch.zeros(2, 128).to(F8), "scale": torch.ones(2, 1)}
    for call in (lambda: ops.add_rms_norm(x, w), lambda: ops.fp8_quantize(x), lambda: ops.fp8_linear(e, e), lambda: ops.fp8_gated(e, e)):
        with pytest.raises(RuntimeError, match="device"):
            call()


def _status(call, make, **kw):
    a = make()
    for f, x in kw.items():
        if isinstance(x, tuple):
            getattr(a, f)[:] = x
        else:
            setattr(a, f, x)
    return call(ctypes.byref(a), None), _lib.load().pkv_last_error()


def _norm():
    a = _lib.NormArgs()
    a.x = a.weight = a.out = 4096
    a.dtype, a.rows, a.width, a.x_stride, a.out_stride = _lib.BF16, 2, 256, 256, 256
    return a


def _quantize():
    a = _lib.Fp8QuantizeArgs()
    a.x = a.codes = a.scale = 4096
    a.x_stride[:], a.codes_stride = (0, 256, 128), 256
    a.dtype, a.rows, a.width, a.per_batch, a.block = _lib.BF16, 2, 256, 2, 1
    return a


def _product():
    a = _lib.Fp8ProductArgs()
    a.x = a.w = a.x_scale = a.w_scale = a.out = 4096
    a.x_stride = a.w_stride = 256
    a.out_stride, a.dtype, a.rows, a.width, a.cols = 32, _lib.F16, 2, 256, 32
    return a


def test_norm_checks_its_arguments():
    call = _lib.load().pkv_add_rms_norm
    assert call(None, None) == _lib.ERR_INVALID
    for kw, code, text in (({"x": None}, "INVALID", b"null"), ({"weight": None}, "INVALID", b"null"), ({"residual": 4096}, "INVALID", b"residual"),
                           ({"sum": 4096}, "INVALID", b"residual"), ({"out": None}, "INVALID", b"result"), ({"codes": 4096, "scale": 4096}, "INVALID", b"result"),
                           ({"out": None, "codes": 4096}, "INVALID", b"result"), ({"scale": 4096}, "INVALID", b"result"), ({"dtype": _lib.F32}, "UNSUPPORTED", b"type"),
                           ({"rows": 0}, "INVALID", b"positive"), ({"width": 0}, "INVALID", b"positive"), ({"width": 24}, "UNSUPPORTED", b"width"),
                           ({"width": 65552}, "UNSUPPORTED", b"width"), ({"rows": 1 << 22}, "UNSUPPORTED", b"rows"), ({"x": 4104}, "INVALID", b"16-byte"),
                           ({"x_stride": 260}, "INVALID", b"16-byte"), ({"out": 4098}, "INVALID", b"16-byte")):
        got, said = _status(call, _norm, **kw)
        assert got == getattr(_lib, "ERR_" + code) and text in said, (kw, got, said)


def test_quantize_checks_its_arguments():
    call = _lib.load().pkv_fp8_quantize
    assert call(None, None) == _lib.ERR_INVALID
    for kw, code, text in (({"x": None}, "INVALID", b"null"), ({"codes": None}, "INVALID", b"null"), ({"scale": None}, "INVALID", b"null"),
                           ({"dtype": _lib.F32}, "UNSUPPORTED", b"type"), ({"rows": 0}, "INVALID", b"positive"), ({"per_batch": 0}, "INVALID", b"positive"),
                           ({"width": 40}, "UNSUPPORTED", b"width"), ({"block": 2}, "UNSUPPORTED", b"blocks"), ({"block": 128, "per_batch": 1}, "UNSUPPORTED", b"heads"),
                           ({"block": 128, "x_stride": (0, 256, 256)}, "UNSUPPORTED", b"heads"), ({"x": 4100}, "INVALID", b"16-byte"),
                           ({"x_stride": (0, 260, 128)}, "INVALID", b"16-byte"), ({"codes_stride": 257}, "INVALID", b"16-byte"),
                           ({"rows": 1 << 30, "per_batch": 1 << 30, "width": 1024}, "UNSUPPORTED", b"too large")):
        got, said = _status(call, _quantize, **kw)
        assert got == getattr(_lib, "ERR_" + code) and text in said, (kw, got, said)


def test_product_checks_its_arguments():
    call = _lib.load().pkv_fp8_product
    assert call(None, None) == _lib.ERR_INVALID
    for f in ("x", "w", "x_scale", "w_scale", "out"):
        assert _status(call, _product, **{f: None})[0] == _lib.ERR_INVALID
    for kw, code, text in (({"dtype": _lib.F32}, "UNSUPPORTED", b"type"), ({"rows": 0}, "INVALID", b"positive"), ({"cols": -1}, "INVALID", b"positive"),
                           ({"width": 200}, "UNSUPPORTED", b"width"), ({"width": (1 << 20) + 16}, "UNSUPPORTED", b"width"), ({"rows": (1 << 24) + 1}, "UNSUPPORTED", b"2^24"),
                           ({"gated": 1, "cols": 24}, "UNSUPPORTED", b"gated"), ({"gated": 1, "bias": 4096}, "UNSUPPORTED", b"gated"), ({"x": 4104}, "INVALID", b"16-byte"),
                           ({"w_stride": 264}, "INVALID", b"16-byte"), ({"x_stride": 128}, "UNSUPPORTED", b"overlap"), ({"w_stride": -256}, "UNSUPPORTED", b"overlap"),
                           ({"x_stride": (1 << 20) + 16}, "UNSUPPORTED", b"2^20"), ({"rows": 1 << 24, "cols": 1 << 24}, "UNSUPPORTED", b"too large")):
        got, said = _status(call, _product, **kw)
        assert got == getattr(_lib, "ERR_" + code) and text in said, (kw, got, said)


def test_product_checks_what_its_numbers_lie_at():
    call = _lib.load().pkv_fp8_product
    for f, at in (("x_scale", 4098), ("w_scale", 4097), ("bias", 4097), ("out", 4097)):
        got, said = _status(call, _product, **{f: at})
        assert got == _lib.ERR_INVALID and b"multiples of their size" in said, (f, got, said)
