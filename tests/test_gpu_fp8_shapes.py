"""The products at the sizes from which each kind of workgroup is chosen on, from 16 x 16 results to 256 x 256, with one block of the width, few and
many, every one of them ragged: bit for bit where sums are exact, and rows and columns of the edges against 64 bits."""
import pytest
import torch

import fp8_oracle as oracle
from packkv_amd import ops

pytestmark = pytest.mark.gpu
# rows of x, width, rows of w.  (What is chosen goes by the rows and columns of tiles and the blocks of the width.)
LINEAR = [(16, 16, 1040), (20, 144, 2064), (33, 656, 1552), (20, 656, 4112), (130, 1040, 1040), (33, 656, 6161), (513, 144, 528), (65, 656, 4112), (257, 144, 1555),
          (97, 656, 4112), (1025, 272, 528), (97, 656, 6160), (1500, 272, 530), (200, 656, 4112), (130, 2064, 6160), (513, 656, 4112), (1025, 1040, 2064),
          (1025, 656, 4113), (700, 144, 6160), (2100, 272, 4112), (1500, 16, 6160), (2100, 656, 4111), (4097, 912, 2070), (97, 1040, 6160), (257, 1040, 3095), (2100, 656, 6160), (3001, 400, 4111),
          (2100, 1040, 6152)]
GATED = [(16, 16, 1040), (20, 656, 2064), (130, 144, 528), (20, 656, 4112), (130, 656, 1040), (33, 656, 4112), (97, 144, 2064), (65, 656, 6160), (257, 272, 2064),
         (200, 656, 4112), (130, 2064, 6160), (513, 656, 4112), (700, 272, 3088), (1025, 656, 4112), (1500, 144, 3088), (2100, 16, 2064), (2500, 912, 2080), (3001, 400, 2064),
         (1500, 656, 6160), (65, 656, 6144), (200, 656, 4096), (1025, 656, 4096), (513, 656, 4096), (2100, 400, 6144), (97, 144, 2048)]          # (whole blocks of 128 last)


def _whole(rows, width, block, gen, cuda):
    down = -(-rows // block)
    codes = torch.randint(-2, 3, (rows, width), generator=gen, device=cuda).float().to(oracle.F8)
    return {"codes": codes, "scale": torch.exp2(torch.randint(-2, 3, (down, -(-width // 128)), generator=gen, device=cuda).float())}


def _drawn(rows, width, block, gen, cuda, size):
    y = size * torch.randn(rows, width, generator=gen, device=cuda) * torch.exp(0.5 * torch.randn(width, generator=gen, device=cuda))
    e = oracle.make_eight(y, block)
    return e


def _some(n, count=24):
    """Rows at both ends, around the borders of tiles, and some between."""
    at = {0, 1, 15, 16, 63, 64, 127, 128, 255, 256, n - 1, n - 2, n // 2, n // 3}
    at |= {int(i * n / count) for i in range(count)}
    return torch.tensor(sorted(i for i in at if 0 <= i < n))


def _part(e, rows, block):
    """Rows of an 8-bit form, a scale for each."""
    rows = rows.to(e["codes"].device)
    return {"codes": e["codes"].view(torch.uint8)[rows].view(oracle.F8), "scale": e["scale"][rows // block]}


@pytest.mark.parametrize("rows,width,cols", LINEAR)
def test_linear(cuda, rows, width, cols):
    gen = torch.Generator(device=cuda).manual_seed(rows + width + cols)
    x, w = _whole(rows, width, 1, gen, cuda), _whole(cols, width, 128, gen, cuda)
    want = (x["codes"].double() * oracle.spread(x["scale"], 1, rows, width)) @ (w["codes"].double() * oracle.spread(w["scale"], 128, cols, width)).t().contiguous()
    assert torch.equal(ops.fp8_linear(x, w), want.to(torch.bfloat16))
    x, w = _drawn(rows, width, 1, gen, cuda, 1.0), _drawn(cols, width, 128, gen, cuda, width ** -0.5)
    bias = torch.randn(cols, generator=gen, device=cuda).half()
    got = ops.fp8_linear(x, w, bias=bias, dtype=torch.float16)
    m, n = _some(rows), _some(cols)
    y, tol, var = oracle.product(_part(x, m, 1), _part(w, n, 128), block=1)
    b = bias.cpu().double()[n]
    oracle.check_rounded(got.cpu()[m][:, n], y + b, tol + oracle.U * (y.abs() + b.abs()), var)


@pytest.mark.parametrize("rows,width,cols", GATED)
def test_gated(cuda, rows, width, cols):
    gen = torch.Generator(device=cuda).manual_seed(rows + width + cols)
    x, w = _drawn(rows, width, 1, gen, cuda, 0.5), _drawn(2 * cols, width, 128, gen, cuda, width ** -0.5)
    got = ops.fp8_gated(x, w, dtype=torch.bfloat16)
    m, n = _some(rows), _some(cols)
    both = [oracle.product(_part(x, m, 1), _part(w, n + at, 128), block=1) for at in (0, cols)]
    oracle.check_rounded(got.cpu()[m][:, n], *oracle.gated(*both))


@pytest.mark.parametrize("rows,width,cols", [(513, 400, 4112), (2100, 144, 4112), (200, 656, 4112)])
def test_nan_rows_between_tiles(cuda, rows, width, cols):
    gen = torch.Generator(device=cuda).manual_seed(rows)
    x, w = _whole(rows, width, 1, gen, cuda), _whole(cols, width, 128, gen, cuda)
    want = ops.fp8_linear(x, w)
    bad_m, bad_n = [0, 128, rows - 1], [1, 255, cols - 1]
    for i in bad_m: x["codes"][i] = float("nan")
    for i in bad_n: w["codes"][i] = float("nan")
    got = ops.fp8_linear(x, w)
    keep = torch.ones(rows, cols, dtype=torch.bool, device=cuda)
    keep[bad_m], keep[:, bad_n] = False, False
    assert torch.equal(got[keep], want[keep]) and bool(torch.isnan(got[~keep]).all())


def test_results_behind_and_beside_stay(cuda):
    """What lies around the result's rows is not written: a call through the C entry into the middle of a larger buffer."""
    import ctypes
    from packkv_amd import _lib
    gen = torch.Generator(device=cuda).manual_seed(1)
    for rows, width, cols, gated in ((5, 144, 33, 0), (130, 272, 2064, 0), (300, 144, 4112, 1), (2100, 144, 4111, 0), (65, 656, 4112, 0)):
        n = cols * (2 if gated else 1)
        x, w = _whole(rows, width, 1, gen, cuda), _whole(n, width, 128, gen, cuda)
        want = ops.fp8_gated(x, w) if gated else ops.fp8_linear(x, w)
        room = torch.full((rows + 2, cols + 24), 7.0, dtype=torch.bfloat16, device=cuda)
        a = _lib.Fp8ProductArgs()
        a.x, a.w, a.x_scale, a.w_scale = (t.data_ptr() for t in (x["codes"], w["codes"], x["scale"], w["scale"]))
        a.out = room[1:, 8:].data_ptr()
        a.x_stride = a.w_stride = width
        a.out_stride = cols + 24
        a.x_scale_stride[:], a.w_scale_stride[:] = x["scale"].stride(), w["scale"].stride()
        a.dtype, a.rows, a.width, a.cols, a.gated = _lib.BF16, rows, width, cols, gated
        _lib.check(_lib.load().pkv_fp8_product(ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
        assert torch.equal(room[1:-1, 8:8 + cols], want)
        room[1:-1, 8:8 + cols] = 7.0
        assert bool((room == 7.0).all())


@pytest.mark.parametrize("rows,width,cols", [(203, 896, 4864), (260, 272, 4096), (700, 144, 4096), (1500, 656, 6144), (1300, 400, 4096)])
def test_gated_where_up_starts_on_a_tile(cuda, rows, width, cols):
    """All rows of a tile's half have one scale: the other half of the kernels' forms at sizes where `GATED` has the ragged one."""
    test_gated(cuda, rows, width, cols)
