"""The 8-bit operators' C entries, called as the framework's own code does not call them."""
import ctypes

import pytest
import torch

import fp8_oracle as oracle
from packkv_amd import _lib, ops

pytestmark = pytest.mark.gpu


def _product(x, w, out, out_stride, rows, cols, gated):
    a = _lib.Fp8ProductArgs()
    a.x, a.w, a.x_scale, a.w_scale, a.out = (t.data_ptr() for t in (x["codes"], w["codes"], x["scale"], w["scale"], out))
    a.x_stride = a.w_stride = width = w["codes"].size(1)
    a.out_stride, a.dtype, a.rows, a.width, a.cols, a.gated = out_stride, _lib.BF16, rows, width, cols, int(gated)
    a.x_scale_stride[:], a.w_scale_stride[:] = x["scale"].stride(), w["scale"].stride()
    _lib.check(_lib.load().pkv_fp8_product(ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))


@pytest.mark.parametrize("width,cols,gated", [(128, 32768, False), (128, 16384, True), (896, 20000, False), (128, 64, False), (128, 64, True)])
def test_a_single_rows_stride_means_nothing(cuda, width, cols, gated):
    """One row of results, with wide ones through the kernel for many rows: the stride to a next row that is not there changes nothing."""
    gen = torch.Generator(device=cuda).manual_seed(cols)
    draw = lambda rows, block: ops.fp8_quantize(torch.randn(rows, width, generator=gen, device=cuda).bfloat16(), block)
    x, w = draw(1, 1), draw((2 if gated else 1) * cols, 128)
    want = ops.fp8_gated(x, w) if gated else ops.fp8_linear(x, w)
    oracle_y, tol, var = oracle.product(x, {f: t[:1] if f == "scale" else t[:128] for f, t in w.items()})
    if not gated:
        oracle.check_rounded(want[:, :128], *(t[:, :cols] for t in (oracle_y, tol, var)))
    for stride in (cols, 0, 8, cols - 8, 3, -8, 1 << 33):
        room = torch.full((cols + 64,), -7.0, dtype=torch.bfloat16, device=cuda)
        _product(x, w, room, stride, 1, cols, gated)
        assert torch.equal(room[:cols], want[0]), stride
        assert bool((room[cols:] == -7).all())
