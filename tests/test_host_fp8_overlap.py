"""Results whose rows or scales lie in one another's memory are refused by the C entries: kernels write rows in any order."""
import ctypes

import pytest

from packkv_amd import _lib


def _status(call, a, kw):
    for f, x in kw.items():
        if isinstance(x, tuple):
            getattr(a, f)[:] = x
        else:
            setattr(a, f, x)
    return call(ctypes.byref(a), None), _lib.load().pkv_last_error()


def _norm(**kw):
    a = _lib.NormArgs()
    a.x = a.weight = 4096
    a.dtype, a.rows, a.width, a.x_stride = _lib.BF16, 5, 400, 400
    return _status(_lib.load().pkv_add_rms_norm, a, kw)


def _quantize(**kw):
    a = _lib.Fp8QuantizeArgs()
    a.x = a.codes = a.scale = 4096
    a.x_stride[:], a.codes_stride = (0, 400, 128), 400
    a.dtype, a.rows, a.width, a.per_batch, a.block = _lib.BF16, 300, 400, 300, 1
    return _status(_lib.load().pkv_fp8_quantize, a, kw)


def _product(**kw):
    a = _lib.Fp8ProductArgs()
    a.x = a.w = a.x_scale = a.w_scale = a.out = 4096
    a.x_stride = a.w_stride = 256
    a.dtype, a.rows, a.width, a.cols = _lib.F16, 2, 256, 32
    return _status(_lib.load().pkv_fp8_product, a, kw)


EIGHT = {"codes": 4096, "scale": 4096, "codes_stride": 400, "scale_stride": (1, 5)}


@pytest.mark.parametrize("call,kw", [
    (_norm, {"out": 4096, "out_stride": 0}), (_norm, {"out": 4096, "out_stride": 392}), (_norm, {"out": 4096, "out_stride": -392}),
    (_norm, {"out": 4096, "out_stride": 400, "residual": 4096, "residual_stride": 400, "sum": 8192, "sum_stride": 8}),
    (_norm, {**EIGHT, "codes_stride": 384}), (_norm, {**EIGHT, "scale_stride": (0, 5)}), (_norm, {**EIGHT, "scale_stride": (1, 4)}),
    (_norm, {**EIGHT, "scale_stride": (3, 1)}), (_norm, {**EIGHT, "scale_stride": (4, 0)}), (_norm, {**EIGHT, "scale_stride": (0, 0)}),
    (_quantize, {"codes_stride": 0, "scale_stride": (1, 300)}), (_quantize, {"codes_stride": 384, "scale_stride": (1, 300)}),
    (_quantize, {"scale_stride": (1, 299)}), (_quantize, {"scale_stride": (0, 0)}), (_quantize, {"scale_stride": (-3, 1)}),
    (_quantize, {"block": 128, "scale_stride": (1, 2)}), (_quantize, {"block": 128, "scale_stride": (0, 1)}),
    (_product, {"out_stride": 0}), (_product, {"out_stride": 31}), (_product, {"out_stride": -31}), (_product, {"out_stride": 31, "gated": 1}),
    (_product, {"out_stride": 8192, "rows": 4000, "cols": 8193}),
])
def test_overlapping_results_are_refused(call, kw):
    got, said = call(**kw)
    assert got == _lib.ERR_INVALID and b"overlap" in said, (got, said)
