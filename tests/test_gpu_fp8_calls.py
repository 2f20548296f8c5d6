"""The ways in which the 8-bit operators can be called: one-dimensional and batched forms, the native host side and the general code, strange
strides, results in an input's place, matrices beyond 4 GiB, graphs replayed side by side, refusals that need a device."""
import ctypes

import pytest
import torch

import fp8_oracle as oracle
from packkv_amd import _lib, ops

pytestmark = pytest.mark.gpu


def _gen(seed, cuda):
    return torch.Generator(device=cuda).manual_seed(seed)


def _same(a, b):
    if isinstance(a, dict):
        assert torch.equal(a["codes"].view(torch.uint8), b["codes"].view(torch.uint8)) and torch.equal(a["scale"], b["scale"])
        assert a["codes"].shape == b["codes"].shape and a["scale"].shape == b["scale"].shape and a["scale"].stride() == b["scale"].stride()
    elif isinstance(a, tuple):
        assert len(a) == len(b)
        for x, y in zip(a, b):
            _same(x, y)
    else:
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_host_side_and_general_code_agree(cuda, monkeypatch):
    gen = _gen(1, cuda)
    x = torch.randn(3, 7, 400, generator=gen, device=cuda).half()
    r = torch.randn(3, 7, 400, generator=gen, device=cuda).half()
    n = torch.rand(400, generator=gen, device=cuda).half()
    a = torch.randn(2, 7, 5, 128, generator=gen, device=cuda).half().transpose(1, 2)
    big = torch.randn(288, 400, generator=gen, device=cuda).half()
    b = torch.randn(288, generator=gen, device=cuda).half()

    def all_of_them():
        e, w = ops.fp8_quantize(x), ops.fp8_quantize(big, 128)
        one = {"codes": e["codes"][1, 2], "scale": e["scale"][1, 2]}
        thin = {"codes": e["codes"][:, 2:3], "scale": e["scale"][:, 2:3]}
        return [ops.add_rms_norm(x, n), ops.add_rms_norm(x, n, 1e-5, r), ops.add_rms_norm(x, n, 1e-5, residual=r, fp8=True), ops.add_rms_norm(x[0, 0], n, fp8=True),
                e, w, ops.fp8_quantize(a, heads=True), ops.fp8_quantize(x[0, 0]), ops.fp8_linear(e, w), ops.fp8_linear(e, w, b, torch.float16),
                ops.fp8_gated(e, w), ops.fp8_linear(one, w), ops.fp8_gated(thin, w, dtype=torch.float16)]

    assert _lib.host is not _lib.NO_HOST
    served = all_of_them()
    monkeypatch.setattr(_lib, "host", _lib.NO_HOST)
    for got, want in zip(served, all_of_them()):
        _same(got, want)


def test_one_dimension_and_none(cuda):
    gen = _gen(2, cuda)
    x = torch.randn(272, generator=gen, device=cuda).bfloat16()
    e = ops.fp8_quantize(x)
    assert e["codes"].shape == (272,) and e["scale"].shape == (3,)
    oracle.check_eight(e, x.cpu().double()[None], 1)
    w = ops.fp8_quantize(torch.randn(40, 272, generator=gen, device=cuda).bfloat16(), 128)
    y, tol, var = oracle.product({"codes": e["codes"][None], "scale": e["scale"][None]}, w)
    assert ops.fp8_linear(e, w).shape == (40,)
    oracle.check_rounded(ops.fp8_linear(e, w), y, tol, var)
    none = ops.fp8_quantize(x.new_empty(0, 272), 128)
    assert none["codes"].shape == (0, 272) and none["scale"].shape == (0, 3)
    assert ops.fp8_linear(e, none).shape == (0,)
    assert ops.fp8_quantize(x.new_empty(4, 0, 272))["scale"].shape == (4, 0, 3)


def test_scales_with_strange_strides(cuda):
    gen = _gen(3, cuda)
    x, w = (ops.fp8_quantize(torch.randn(m, 400, generator=gen, device=cuda).half(), b) for m, b in ((5, 1), (260, 128)))
    want = ops.fp8_linear(x, w)
    room = torch.empty(5, (1 << 20) + 64, device=cuda)
    far = room[:, 7:7 + 2 * x["scale"].size(1):2].copy_(x["scale"])
    assert torch.equal(ops.fp8_linear({"codes": x["codes"], "scale": far}, w), want)
    far_w = room[:3, 1000:1000 + w["scale"].size(1)].copy_(w["scale"])
    assert torch.equal(ops.fp8_linear(x, {"codes": w["codes"], "scale": far_w}), want)
    for i in (0, 4):                                       # one row, whose stride means nothing
        one = {"codes": x["codes"][i:i + 1], "scale": torch.as_strided(far, (1, far.size(1)), (1 << 30, 2), far.storage_offset() + i * far.stride(0))}
        assert torch.equal(ops.fp8_linear(one, w), want[i:i + 1])
    same = {"codes": x["codes"][:1].expand(300, 400), "scale": x["scale"][:1].expand(300, 4)}
    assert torch.equal(ops.fp8_linear(same, w).half(), want[:1].expand(300, 260).half())
    spread = {"codes": x["codes"].new_empty(5, 3, 400).copy_(x["codes"][:, None]).transpose(0, 1), "scale": x["scale"][None].expand(3, 5, 4)}
    assert torch.equal(ops.fp8_linear(spread, w), want.expand(3, 5, 260))


def test_the_sum_in_the_residuals_place(cuda):
    gen = _gen(4, cuda)
    for rows, width in ((1, 4096), (1500, 528), (3, 20000)):
        x, r = (torch.randn(rows, width, generator=gen, device=cuda).bfloat16() for _ in range(2))
        w = torch.rand(width, generator=gen, device=cuda).bfloat16()
        y, h = ops.add_rms_norm(x, w, residual=r)
        a = _lib.NormArgs()
        out = torch.empty_like(x)
        a.x, a.residual, a.sum, a.weight, a.out = x.data_ptr(), r.data_ptr(), r.data_ptr(), w.data_ptr(), out.data_ptr()
        a.x_stride = a.residual_stride = a.sum_stride = a.out_stride = width
        a.dtype, a.rows, a.width, a.eps = _lib.BF16, rows, width, 1e-6
        _lib.check(_lib.load().pkv_add_rms_norm(ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
        assert torch.equal(out, y) and torch.equal(r, h)


def test_weights_beyond_4_gib(cuda):
    gen = _gen(5, cuda)
    rows, width = (1 << 20) + 4000, 4112
    assert rows * width > 1 << 32
    w = {"codes": torch.zeros(rows, width, dtype=torch.uint8, device=cuda).view(oracle.F8), "scale": torch.ones(-(-rows // 128), 33, device=cuda)}
    at = torch.tensor([0, 5, (1 << 32) // width - 1, (1 << 32) // width, (1 << 32) // width + 1, rows - 1], device=cuda)
    part = torch.randint(-2, 3, (at.numel(), width), generator=gen, device=cuda).float().to(oracle.F8)
    w["codes"].view(torch.uint8)[at] = part.view(torch.uint8)
    for m in (1, 40):
        x = {"codes": torch.randint(-2, 3, (m, width), generator=gen, device=cuda).float().to(oracle.F8), "scale": torch.ones(m, 33, device=cuda)}
        got = ops.fp8_linear(x, w)
        want = (x["codes"].double() @ part.double().t().contiguous()).bfloat16()
        assert torch.equal(got[:, at], want)
        got[:, at] = 0
        assert not bool(got.any())
        if m == 1:
            gated = ops.fp8_gated(x, w)
            assert gated.shape == (1, rows // 2) and not bool(gated.any())           # (a gate or an up of zero everywhere)


def test_activations_beyond_4_gib(cuda):
    gen = _gen(6, cuda)
    rows, width = (1 << 20) + 1500, 4112
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=cuda)
    at = torch.tensor([0, (1 << 31) // width, (1 << 32) // width, rows - 1], device=cuda)
    x[at] = torch.randn(at.numel(), width, generator=gen, device=cuda).bfloat16()
    n = torch.ones(width, dtype=torch.bfloat16, device=cuda)
    some = x[at]
    e = ops.fp8_quantize(x)
    _part = lambda e: {"codes": e["codes"].view(torch.uint8)[at].view(oracle.F8), "scale": e["scale"][at]}
    oracle.check_eight(_part(e), some.cpu().double(), 1)
    w = ops.fp8_quantize(torch.randn(48, width, generator=gen, device=cuda).bfloat16(), 128)
    got = ops.fp8_linear(e, w)
    oracle.check_rounded(got[at], *oracle.product(_part(e), w))
    got[at] = 0
    assert not bool(got.any())
    del e, got
    b = ops.fp8_quantize(x, 128)
    codes = b["codes"].view(torch.uint8)
    for i in at.tolist():
        block = x[i // 128 * 128:i // 128 * 128 + 128]
        alone = ops.fp8_quantize(block, 128)
        assert torch.equal(codes[i // 128 * 128:i // 128 * 128 + 128], alone["codes"].view(torch.uint8)) and torch.equal(b["scale"][i // 128], alone["scale"][0])
    del b, codes
    y = ops.add_rms_norm(x, n, fp8=True)
    got = _part(y)
    want = some.cpu().double() / torch.sqrt(some.cpu().double().square().mean(-1, keepdim=True) + 1e-6)
    oracle.check_eight(got, want, 1, 52 * oracle.U)          # (test_gpu_fp8.py's bound)


def test_graphs_side_by_side(cuda):
    """Two captured runs of the layer's operators, replayed on two streams at once: nothing is shared between them."""
    gen = _gen(7, cuda)
    w1 = ops.fp8_quantize(torch.randn(1024, 512, generator=gen, device=cuda).bfloat16() / 20, 128)
    w2 = ops.fp8_quantize(torch.randn(512, 512, generator=gen, device=cuda).bfloat16() / 20, 128)
    n = torch.ones(512, dtype=torch.bfloat16, device=cuda)
    xs = [torch.randn(m, 512, generator=gen, device=cuda).bfloat16() for m in (3, 200)]

    def run(x):
        y, h = ops.add_rms_norm(x, n, residual=x, fp8=True)
        return ops.fp8_linear(ops.fp8_quantize(ops.fp8_gated(y, w1)), w2), h

    for x in xs:
        run(x)
    torch.cuda.synchronize()
    graphs = []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = run(x)
        graphs.append((g, held))
    streams = [torch.cuda.Stream() for _ in xs]
    for seed in range(3):
        for x in xs:
            x.copy_(torch.randn(x.shape, generator=_gen(seed, cuda), device=cuda))
        want = [run(x) for x in xs]
        torch.cuda.synchronize()
        for _ in range(4):
            for (g, _), s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for (_, held), y in zip(graphs, want):
            _same(held, y)


def test_refusals(cuda):
    h = lambda *shape: torch.zeros(*shape, dtype=torch.float16, device=cuda)
    f8 = lambda *shape: torch.zeros(*shape, device=cuda).to(oracle.F8)
    f32 = lambda *shape: torch.ones(*shape, device=cuda)
    e, w = {"codes": f8(4, 256), "scale": f32(4, 2)}, {"codes": f8(64, 256), "scale": f32(1, 2)}
    bad = [
        (lambda: ops.add_rms_norm(h(2, 24), h(24)), "width"), (lambda: ops.add_rms_norm(h(2, 65552), h(65552)), "width"),
        (lambda: ops.add_rms_norm(h(2, 32).float(), h(32)), "Unsupported data type"), (lambda: ops.add_rms_norm(h(2, 32), h(16)), "weight"),
        (lambda: ops.add_rms_norm(h(2, 32), h(32).bfloat16()), "weight"), (lambda: ops.add_rms_norm(h(2, 32), h(32), residual=h(3, 32)), "residual"),
        (lambda: ops.add_rms_norm(h(2, 32), h(32), residual=h(2, 32).bfloat16()), "residual"), (lambda: ops.add_rms_norm(h(2, 32), h(32).cpu()), "weight"),
        (lambda: ops.fp8_quantize(h(2, 40)), "width"), (lambda: ops.fp8_quantize(h(2, 32), block=64), "not supported"),
        (lambda: ops.fp8_quantize(h(2, 2, 32), block=128), "not supported"), (lambda: ops.fp8_quantize(h(2, 32).float()), "Unsupported"),
        (lambda: ops.fp8_quantize(h(2, 3, 64), heads=True), "heads"), (lambda: ops.fp8_quantize(h(1, 2, 3, 64), heads=True), "heads"),
        (lambda: ops.fp8_quantize(h(2, 3, 4, 128), block=128, heads=True), "not supported"),
        (lambda: ops.fp8_linear(h(4, 256), w), "8-bit forms"), (lambda: ops.fp8_linear(e, h(4, 256)), "8-bit forms"), (lambda: ops.fp8_linear({}, w), "8-bit forms"),
        (lambda: ops.fp8_linear({"codes": f8(4, 128), "scale": f32(4, 1)}, w), "width"),
        (lambda: ops.fp8_linear({"codes": e["codes"], "scale": f32(4, 1)}, w), "scales"), (lambda: ops.fp8_linear(e, {"codes": w["codes"], "scale": f32(2, 2)}), "scales"),
        (lambda: ops.fp8_linear({"codes": e["codes"].view(torch.uint8), "scale": e["scale"]}, w), "float8"),
        (lambda: ops.fp8_linear({"codes": e["codes"], "scale": e["scale"].half()}, w), "float32"), (lambda: ops.fp8_linear(e, w, dtype=torch.float32), "Unsupported"),
        (lambda: ops.fp8_linear(e, w, bias=h(64)), "bias"), (lambda: ops.fp8_linear(e, w, bias=h(63).bfloat16()), "bias"),
        (lambda: ops.fp8_linear(e, {"codes": w["codes"].cpu(), "scale": w["scale"]}), "one device"),
        (lambda: ops.fp8_gated(e, {"codes": f8(48, 256), "scale": f32(1, 2)}), "gate and up"),
        (lambda: ops.fp8_linear({"codes": f8(4, 200), "scale": f32(4, 2)}, {"codes": f8(64, 200), "scale": f32(1, 2)}), "width 200"),
    ]
    for call, text in bad:
        with pytest.raises(RuntimeError, match=text):
            call()


def test_sizes_past_an_int_are_refused(cuda):
    """Not taken for what is left of them in 32 bits: 2^32 + 4 rows (one row, repeated) for 4, a width of 2^32 + 16 for 16."""
    rows = (1 << 32) + 4
    h, one = torch.zeros(1, 16, dtype=torch.float16, device=cuda), torch.ones(16, dtype=torch.float16, device=cuda)
    e = lambda n, f: {"codes": h.to(oracle.F8).expand(n, 16), "scale": torch.ones(1, 1, device=cuda).expand(f, 1)}
    for call, text in ((lambda: ops.add_rms_norm(h.expand(rows, 16), one), "rows"), (lambda: ops.add_rms_norm(h.expand(1 << 22, 16), one, fp8=True), "rows"),
                       (lambda: ops.fp8_quantize(h.expand(rows, 16)), "too large"), (lambda: ops.fp8_quantize(h.expand(rows, 16), block=128), "too large"),
                       (lambda: ops.fp8_quantize(torch.empty(1, 1, 1, 128, dtype=torch.float16, device=cuda).expand(1 << 20, 1, 1 << 12, 128), heads=True), "too large"),
                       (lambda: ops.fp8_quantize(torch.empty((1 << 32) + 16, dtype=torch.float16, device=cuda)), "too large"),
                       (lambda: ops.fp8_linear(e(rows, rows), e(16, 1)), "2^24"), (lambda: ops.fp8_linear(e(2, 2), e(rows, (rows + 127) // 128)), "2^24"),
                       (lambda: ops.fp8_gated(e(2, 2), e(rows + 28, (rows + 28 + 127) // 128)), "2^24")):
        with pytest.raises(RuntimeError, match=text.replace("^", "\\^")):
            call()
