"""add_rms_norm, fp8_quantize, fp8_linear and fp8_gated against their definitions in 64 bits (fp8_oracle.py derives the tolerances).

The norm in fp32: a row's sum of squares is at most 64 products in a chain, six joins of a wavefront, sixteen of wavefronts, on values that the
residual's sum rounded once: below 90 roundings, halved by the root; mean, eps, root, reciprocal, two products, the sum: 52 roundings at most."""
import pytest
import torch

import fp8_oracle as oracle
from packkv_amd import ops

pytestmark = pytest.mark.gpu
NORM_REL = 52 * oracle.U
TYPES = [torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _values(rows, width, gen, loud=True):
    x = torch.randn(rows, width, generator=gen) * torch.exp(0.5 * torch.randn(width, generator=gen))
    if loud:
        x[:, torch.randint(0, width, (max(1, width // 200),), generator=gen)] *= 20
    return x


def _eight(rows, width, block, gen, cuda, size=1.0):
    e = oracle.make_eight(size * _values(rows, width, gen, block == 1), block)
    return {"codes": e["codes"].to(cuda), "scale": e["scale"].to(cuda)}


def _check_norm(x, w, eps, res, y, h, dtype, fp8):
    hd = x.cpu().double() + (res.cpu().double() if res is not None else 0)
    hd = hd.reshape(-1, x.size(-1))
    if res is not None:
        assert h.dtype == dtype and h.shape == x.shape
        err = (h.cpu().double().reshape(hd.shape) - hd).abs()
        assert bool((err <= (oracle.half_step(dtype) + 2 * oracle.U) * hd.abs() + oracle.tiny(dtype)).all())
    want = hd / torch.sqrt(hd.square().mean(-1, keepdim=True) + eps) * w.cpu().double()
    if fp8:
        assert y["codes"].shape == x.shape and y["scale"].shape == (*x.shape[:-1], -(-x.size(-1) // 128))
        oracle.check_eight(y, want, 1, NORM_REL)
    else:
        assert y.dtype == dtype and y.shape == x.shape
        err = (y.cpu().double().reshape(want.shape) - want).abs()
        assert bool((err <= (oracle.half_step(dtype) * (1 + NORM_REL) + NORM_REL) * want.abs() + oracle.tiny(dtype)).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,residual", [(1, 4096, True), (1, 16, False), (3, 912, True), (5, 128, False), (2, 8208, True), (7, 144, True), (2, 16400, False),
                                                 (1, 65536, True), (1, 33000 // 16 * 16, True), (1025, 64, True), (1300, 528, False), (1030, 1040, True),
                                                 (1024, 2064, True), (1027, 4096, False), (77, 5120, True), (1100, 4112, True)])
def test_norm_follows_the_formula(cuda, dtype, rows, width, residual):
    gen = _gen(rows + width)
    x = _values(rows, width, gen).to(dtype).to(cuda)
    res = (3 * _values(rows, width, gen)).to(dtype).to(cuda) if residual else None
    w = (1 + 0.3 * torch.randn(width, generator=gen)).to(dtype).to(cuda)
    for fp8 in (False, True):
        got = ops.add_rms_norm(x, w, 1e-5, residual=res, fp8=fp8)
        y, h = got if residual else (got, None)
        _check_norm(x, w, 1e-5, res, y, h, dtype, fp8)


def test_norm_of_strided_rows_and_batches(cuda):
    gen = _gen(5)
    big = _values(2 * 3, 1024, gen).to(torch.bfloat16).to(cuda).view(2, 3, 1024)
    w = torch.ones(264, dtype=torch.bfloat16, device=cuda)[8:].contiguous()
    x, res = big[:, :, 256:512], big[:, :, 512:768]
    y, h = ops.add_rms_norm(x, w, residual=res, fp8=True)
    _check_norm(x, w, 1e-6, res, y, h, torch.bfloat16, True)
    odd = big[:, :, 1:257]                                 # rows off the 16-byte boundaries
    _check_norm(odd, w, 1e-6, None, ops.add_rms_norm(odd, w), None, torch.bfloat16, False)
    one = big[0, 0, 256:512]
    _check_norm(one, w, 1e-6, None, ops.add_rms_norm(one, w), None, torch.bfloat16, False)
    same = x[:, :1].expand(2, 3, 256)
    _check_norm(same, w, 1e-6, None, ops.add_rms_norm(same, w), None, torch.bfloat16, False)
    none = ops.add_rms_norm(x[:, :0], w, residual=res[:, :0], fp8=True)
    assert none[0]["codes"].shape == (2, 0, 256) and none[0]["scale"].shape == (2, 0, 2) and none[1].shape == (2, 0, 256)


def test_norm_of_zeroes_and_of_rows_that_are_not_finite(cuda):
    x = torch.zeros(4, 256, dtype=torch.float16, device=cuda)
    x[1, 3], x[2, 200] = float("nan"), float("inf")
    x[3] = 60000.0
    w = torch.ones(256, dtype=torch.float16, device=cuda)
    e = ops.add_rms_norm(x, w, fp8=True)
    c = e["codes"].float().cpu()
    assert bool((c[0] == 0).all()) and bool(torch.isnan(c[1]).all()) and bool((c[3] == 448).all())
    assert bool(torch.isnan(c[2, 200])) and bool((c[2, :200] == 0).all())              # infinity / infinity
    s = e["scale"].cpu().double()
    assert bool((s[0] == s[1]).all()) and abs(s[0, 0].item() * 448 / oracle.LEAST - 1) < 1e-6 and bool(torch.isfinite(s).all())
    # a sum beyond fp16: the stored sum is infinite, its norm is not
    y, h = ops.add_rms_norm(x[3:], w, residual=x[3:])
    assert bool(torch.isinf(h).all()) and bool((y == 1).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,block", [(1, 16, 1), (1, 16, 128), (3, 4096, 1), (67, 912, 1), (129, 144, 1), (127, 144, 128), (128, 128, 128),
                                              (257, 1168, 128), (1, 8192, 128), (300, 128, 1)])
def test_quantize_follows_the_formula(cuda, dtype, rows, width, block):
    gen = _gen(rows * width + block)
    x = _values(rows, width, gen)
    x[0, :16] = 0
    if rows > 2:
        x[1] *= 1e-3
        x[2, :: 3] = 0
    x = x.to(dtype).to(cuda)
    e = ops.fp8_quantize(x, block=block)
    assert e["codes"].dtype == torch.float8_e4m3fn and e["scale"].dtype == torch.float32
    oracle.check_eight(e, x.cpu().double(), block)


def test_quantize_of_values_that_are_not_finite(cuda):
    x = torch.randn(5, 300 // 16 * 16, generator=_gen(3)).to(torch.bfloat16)
    x[0, 5], x[1, 130], x[2, 131], x[3, 0], x[3, 1] = float("nan"), float("inf"), -float("inf"), 3e38, 1e-38
    x[4] = 1e-39                                           # below the smallest scale: zeroes
    for block in (1, 128):
        e = ops.fp8_quantize(x.to(cuda), block=block)
        oracle.check_eight(e, x.double(), block)
        assert bool(torch.isfinite(e["scale"]).all())


def test_quantize_of_attention_heads_and_strides(cuda):
    gen = _gen(9)
    a = torch.randn(2, 5, 7, 128, generator=gen).to(torch.float16).to(cuda)                   # [B, H, n, 128]
    want = a.transpose(1, 2).reshape(2, 7, 640)
    laid = a.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.empty(2, 5, 7, 136, dtype=torch.float16, device=cuda)[..., 4:132].copy_(a)
    for x in (a, laid, odd):
        e = ops.fp8_quantize(x, heads=True)
        plain = ops.fp8_quantize(want)
        assert e["codes"].shape == (2, 7, 640) and e["scale"].shape == (2, 7, 5)
        assert torch.equal(e["codes"].view(torch.uint8), plain["codes"].view(torch.uint8)) and torch.equal(e["scale"], plain["scale"])
    oracle.check_eight(plain, want.cpu().double().reshape(14, 640), 1)
    one = a[:, :, :1]
    e = ops.fp8_quantize(one, heads=True)
    assert torch.equal(e["codes"].view(torch.uint8), plain["codes"][:, :1].view(torch.uint8)) and torch.equal(e["scale"], plain["scale"][:, :1])
    none = ops.fp8_quantize(a[:, :, :0], heads=True)
    assert none["codes"].shape == (2, 0, 640) and none["scale"].shape == (2, 0, 5)
    cut = want[:, 1:5, 128:512]
    oracle.check_eight(ops.fp8_quantize(cut), cut.cpu().double().reshape(8, 384), 1)
    tall = want.view(14, 640)[:, 16:400]
    oracle.check_eight(ops.fp8_quantize(tall, block=128), tall.cpu().double(), 128)


SHAPES = [(1, 16, 1), (1, 128, 16), (1, 4096, 64), (2, 48, 17), (15, 144, 129), (16, 256, 100), (17, 1040, 33), (33, 896, 160), (48, 512, 200), (64, 128, 257),
          (65, 272, 96), (130, 640, 130), (300, 1152, 272), (257, 400, 513)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,cols", SHAPES)
def test_linear_follows_the_formula(cuda, dtype, rows, width, cols):
    gen = _gen(rows + width + cols)
    x, w = _eight(rows, width, 1, gen, cuda), _eight(cols, width, 128, gen, cuda, width ** -0.5)
    y, tol, var = oracle.product(x, w)
    got = ops.fp8_linear(x, w, dtype=dtype)
    assert got.dtype == dtype and got.shape == (rows, cols)
    oracle.check_rounded(got, y, tol, var)
    bias = torch.randn(cols, generator=gen).to(dtype).to(cuda)
    b = bias.cpu().double()
    oracle.check_rounded(ops.fp8_linear(x, w, bias=bias, dtype=dtype), y + b, tol + oracle.U * (y.abs() + b.abs()), var)


@pytest.mark.parametrize("rows,width,cols", SHAPES + [(700, 336, 777), (1024, 128, 384), (513, 2064, 260)])
def test_linear_of_whole_numbers_is_exact(cuda, rows, width, cols):
    """Codes -2 .. 2 and scales that are powers of two: no product is cut and every sum is exact, so each result is the sum's nearest bf16."""
    gen = _gen(rows * cols + width)
    whole = lambda *shape: torch.randint(-2, 3, shape, generator=gen).float().to(oracle.F8).to(cuda)
    power = lambda *shape: torch.exp2(torch.randint(-2, 3, shape, generator=gen).float()).to(cuda)
    blocks = -(-width // 128)
    x, w = {"codes": whole(rows, width), "scale": power(rows, blocks)}, {"codes": whole(cols, width), "scale": power(-(-cols // 128), blocks)}
    y, _, _ = oracle.product({f: t[:, :] for f, t in x.items()}, w) if rows * cols * width < 1 << 24 else (None, None, None)
    if y is None:
        xd = x["codes"].cpu().double() * oracle.spread(x["scale"].cpu(), 1, rows, width)
        y = xd @ (w["codes"].cpu().double() * oracle.spread(w["scale"].cpu(), 128, cols, width)).t()
    assert torch.equal(ops.fp8_linear(x, w).cpu(), y.to(torch.bfloat16))
    if cols % 32 == 0:
        g, u = y[:, :cols // 2], y[:, cols // 2:]
        got = ops.fp8_gated(x, w, dtype=torch.float16).cpu().double()
        want = g * torch.sigmoid(g) * u
        inside = want.abs() < 65000
        err = ((got - want).abs() - (2.0 ** -11 + 2 * oracle.U * (g.abs() + 8)) * want.abs() - 2.0 ** -25)[inside]
        assert bool((err <= 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,cols", [(1, 16, 16), (1, 4096, 48), (3, 144, 144), (16, 256, 112), (33, 896, 160), (64, 384, 272), (129, 640, 144), (300, 400, 528)])
def test_gated_follows_the_formula(cuda, dtype, rows, width, cols):
    gen = _gen(rows + width * cols)
    x, w = _eight(rows, width, 1, gen, cuda, 0.5), _eight(2 * cols, width, 128, gen, cuda, width ** -0.5)
    y, tol, var = oracle.product(x, w)
    half = lambda t: (t[:, :cols], t[:, cols:])
    (g, u), (tg, tu), (vg, vu) = half(y), half(tol), half(var)
    got = ops.fp8_gated(x, w, dtype=dtype)
    assert got.dtype == dtype and got.shape == (rows, cols)
    oracle.check_rounded(got, *oracle.gated((g, tg, vg), (u, tu, vu)))


def test_product_reads_scales_and_codes_where_they_lie(cuda):
    gen = _gen(11)
    x, w = _eight(21, 400, 1, gen, cuda), _eight(150, 400, 128, gen, cuda)
    want = ops.fp8_linear(x, w)
    turned = lambda e: {"codes": e["codes"], "scale": e["scale"].t().contiguous().t()}
    wide = lambda e: {"codes": torch.zeros(e["codes"].size(0), 512, device=cuda).to(oracle.F8)[:, 64:464].copy_(e["codes"]), "scale": e["scale"]}
    off = lambda e: {"codes": torch.zeros(e["codes"].size(0), 512, device=cuda).to(oracle.F8)[:, 3:403].copy_(e["codes"]), "scale": e["scale"]}
    for a in (turned, wide, off):
        for b in (turned, wide, off):
            assert torch.equal(ops.fp8_linear(a(x), b(w)), want)
    batch = {"codes": x["codes"].view(3, 7, 400), "scale": x["scale"].view(3, 7, 4)}
    assert torch.equal(ops.fp8_linear(batch, w), want.view(3, 7, 150))
    part = {"codes": batch["codes"][:, 2:5], "scale": batch["scale"][:, 2:5]}
    assert torch.equal(ops.fp8_linear(part, w), want.view(3, 7, 150)[:, 2:5])
    alone = {"codes": x["codes"][4], "scale": x["scale"][4]}
    assert torch.equal(ops.fp8_linear(alone, w), want[4])
    same = {"codes": x["codes"][:1].expand(21, 400), "scale": x["scale"][:1].expand(21, 4)}
    assert torch.equal(ops.fp8_linear(same, w), want[:1].expand(21, 150))
    none = {"codes": x["codes"][:0], "scale": x["scale"][:0]}
    assert ops.fp8_linear(none, w).shape == (0, 150)


@pytest.mark.parametrize("rows", [1, 5, 40, 200, 600])
def test_a_row_of_nan_stays_in_its_row(cuda, rows):
    """NaN codes behind a row's ragged end belong to the next row, and do not reach this one; nor does a NaN row of w other results."""
    gen = _gen(rows)
    x, w = _eight(rows, 144, 1, gen, cuda), _eight(160, 144, 128, gen, cuda)
    want = ops.fp8_linear(x, w)
    x["codes"][rows // 2] = float("nan")
    w["codes"][70] = float("nan")
    got = ops.fp8_linear(x, w)
    assert bool(torch.isnan(got[rows // 2]).all()) and bool(torch.isnan(got[:, 70]).all())
    keep = torch.ones(rows, 160, dtype=torch.bool)
    keep[rows // 2], keep[:, 70] = False, False
    assert torch.equal(got.cpu()[keep], want.cpu()[keep])


def test_results_do_not_depend_on_the_batch(cuda):
    """A row alone, and the same row among few and many, to the last rounding's tolerance; the same call again bit for bit."""
    gen = _gen(2)
    x, w = _eight(700, 1024, 1, gen, cuda), _eight(384, 1024, 128, gen, cuda, 1 / 32)
    want = ops.fp8_linear(x, w, dtype=torch.float16)
    assert torch.equal(ops.fp8_linear(x, w, dtype=torch.float16), want)
    y, tol, var = oracle.product({f: t[:3] for f, t in x.items()}, w)
    for n in (1, 3, 20, 100, 300):
        got = ops.fp8_linear({f: t[:n] for f, t in x.items()}, w, dtype=torch.float16)
        m = min(n, 3)
        oracle.check_rounded(got[:m], y[:m], tol[:m], var[:m])


def test_other_streams_and_graphs(cuda):
    gen = _gen(8)
    w1, w2 = _eight(2 * 256, 512, 128, gen, cuda, 1 / 23), _eight(512, 256, 128, gen, cuda, 1 / 16)
    norm = torch.ones(512, dtype=torch.bfloat16, device=cuda)
    x = torch.randn(9, 512, generator=gen).to(torch.bfloat16).to(cuda)
    h = torch.randn(9, 512, generator=gen).to(torch.bfloat16).to(cuda)

    def block():
        y, s = ops.add_rms_norm(x, norm, residual=h, fp8=True)
        return ops.fp8_linear(ops.fp8_quantize(ops.fp8_gated(y, w1)), w2), s

    want = block()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = block()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = block()
    for seed in range(3):
        x.copy_(torch.randn(9, 512, generator=_gen(seed)).to(torch.bfloat16))
        graph.replay()
        want = block()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
