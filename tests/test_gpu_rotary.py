"""norm_rotary and window_append_rotary against the formula in 64 bits.

Tolerance, per element: half a step of the stored type, and what the kernel's 32-bit steps lose of the two channels a and b that
meet in it.  The sum of squares is 128 products in chains of 16 and three joins (20 roundings, halved by the root), mean, eps, root,
reciprocal, two products and the turn's four more: below 24 roundings of 2^-24; the fraction of a turn is rounded once to 24 bits
(at most 2^-26 turns, 2 pi 2^-26 < 2 * 2^-24 radians) and the library's sine and cosine add 2 steps (4 halves).  32 * 2^-24 * (|a| + |b|)."""
import numpy as np
import pytest
import torch

from packkv_amd import ops

pytestmark = pytest.mark.gpu
FAR = 1 << 40


def _inv(cuda, theta=1.0e6):
    return 1.0 / (theta ** (torch.arange(0, 128, 2, device=cuda, dtype=torch.float32) / 128))


def _formula(x, w, pos, inv, axis, eps):
    """(result, |a| + |b| of each channel's pair) in 64 bits on the CPU; pos [A, B, n]."""
    x = x.cpu().double()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.cpu().double()
    # (a position of 40 bits times a frequency of 24 fills the 64 bits of an extended double; 53 would be off by 6e-5 there)
    angle = np.moveaxis(pos.cpu().numpy().astype(np.longdouble)[list(axis)], 0, -1) * inv.cpu().numpy().astype(np.longdouble)
    c, s = (torch.from_numpy(f(angle).astype(np.float64))[:, None] for f in (np.cos, np.sin))
    a, b = x[..., :64], x[..., 64:]
    size = a.abs() + b.abs()
    return torch.cat((a * c - b * s, b * c + a * s), -1), torch.cat((size, size), -1)


def _check(got, x, w, pos, inv, axis, eps=1e-6):
    want, size = _formula(x, w, pos, inv, axis, eps)
    half = torch.finfo(got.dtype).eps / 2
    tol = half * want.abs() + torch.finfo(got.dtype).smallest_normal * half + 32 * 2.0 ** -24 * size
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol * (1 + half)).all()), (err.max().item(), (err / tol).max().item())


def _pos(cuda, B, n, far, A, gen):
    base = torch.randint(0, far + 1, (1, B, 1), generator=gen, device=cuda) + torch.arange(n, device=cuda)
    return base + (torch.randint(0, 99, (A, B, n), generator=gen, device=cuda) if A > 1 else 0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Hq,Hkv,n,sections,inter,far,norm", [
    (1, 1, 1, 1, None, False, 0, True), (2, 32, 8, 5, None, False, 1000000, True), (3, 14, 2, 33, (16, 24, 24), False, 5000, True),
    (1, 40, 9, 2, (24, 20, 20), True, FAR, False), (2, 7, 7, 129, (64,), False, 100, False), (1, 32, 32, 3, (30, 20, 10, 4), False, 70000, True)])
def test_norm_rotary_follows_the_formula(cuda, dtype, B, Hq, Hkv, n, sections, inter, far, norm):
    gen = torch.Generator(device=cuda).manual_seed(n)
    qkv = (torch.randn(B, n, Hq + Hkv, 128, generator=gen, device=cuda) * 3).to(dtype)
    q, k = qkv[:, :, :Hq].transpose(1, 2), qkv[:, :, Hq:].transpose(1, 2)
    w = [(1 + 0.3 * torch.randn(128, generator=gen, device=cuda)).to(dtype) if norm else None for _ in range(2)]
    A = 1 if sections is None else len(sections)
    pos, inv = _pos(cuda, B, n, far, A, gen), _inv(cuda)
    gq, gk = ops.norm_rotary(q, k, pos[0] if sections is None else pos, inv, w[0], w[1], sections=sections, interleaved=inter)
    assert gq.shape == q.shape and gk.shape == k.shape and gq.is_contiguous() and gk.is_contiguous() and gq.dtype == dtype
    axis = ops._frequency_axes(sections, inter)
    _check(gq, q, w[0], pos, inv, axis)
    _check(gk, k, w[1], pos, inv, axis)


def test_the_largest_prompts_and_one_weight_only(cuda):
    gen = torch.Generator(device=cuda).manual_seed(3)
    q = torch.randn(4, 32, 2048, 128, generator=gen, device=cuda).bfloat16()
    k = torch.randn(4, 8, 2048, 128, generator=gen, device=cuda).bfloat16()
    w = (1 + 0.3 * torch.randn(128, generator=gen, device=cuda)).bfloat16()
    pos, inv = _pos(cuda, 4, 2048, 32768, 1, gen), _inv(cuda)
    for qw, kw in ((w, None), (None, w)):
        gq, gk = ops.norm_rotary(q, k, pos[0], inv, qw, kw, eps=1e-5)
        _check(gq, q, qw, pos, inv, bytes(64), 1e-5)
        _check(gk, k, kw, pos, inv, bytes(64), 1e-5)


def test_layouts_types_of_positions_and_rows_without_alignment(cuda):
    """Rows at odd addresses, heads shared by expansion, int32 and broadcast positions: as contiguous copies give."""
    gen = torch.Generator(device=cuda).manual_seed(4)
    inv = _inv(cuda)
    flat = torch.randn(2 * 9 * 6 * 131 + 3, generator=gen, device=cuda).half()
    odd = flat[3:].as_strided((2, 6, 9, 128), (9 * 6 * 131, 131, 6 * 131, 1))
    one = torch.randn(2, 1, 9, 128, generator=gen, device=cuda).half().expand(2, 5, 9, 128)
    pos = _pos(cuda, 2, 9, 3000, 1, gen)[0]
    want = ops.norm_rotary(odd.contiguous(), one.contiguous(), pos, inv)
    got = ops.norm_rotary(odd, one, pos.int(), inv)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    turned = odd.transpose(2, 3).contiguous().transpose(2, 3)          # channels not adjacent
    assert torch.equal(ops.norm_rotary(turned, one, pos, inv)[0], want[0])
    row = pos[:1]
    want = ops.norm_rotary(odd, one, row.expand(2, 9).contiguous(), inv)
    for same in (row, row[0]):
        assert all(torch.equal(a, b) for a, b in zip(ops.norm_rotary(odd, one, same, inv), want))
    want = ops.norm_rotary(odd, one, pos, inv)
    three = ops.norm_rotary(odd, one, pos[None].expand(3, 2, 9), inv, sections=(16, 24, 24))
    assert all(torch.equal(a, b) for a, b in zip(three, want))


def test_rows_of_zeros_infinities_and_nothing_at_all(cuda):
    inv = _inv(cuda)
    w = torch.ones(128, device=cuda).half()
    x = torch.zeros(1, 3, 1, 128, device=cuda).half()
    x[0, 1, 0, 5] = float("nan")
    x[0, 2, 0, 64] = 65504.0
    got, _ = ops.norm_rotary(x, x, torch.zeros(1, 1, dtype=torch.int64, device=cuda), inv, w, w)
    assert bool((got[0, 0] == 0).all()) and bool(got[0, 1].isnan().all())
    assert abs(got[0, 2, 0, 64].item() - 128 ** 0.5) < 0.01 and int((got[0, 2] != 0).sum()) == 1
    empty = torch.zeros(2, 3, 0, 128, device=cuda).half()
    a, b = ops.norm_rotary(empty, empty, torch.zeros(2, 0, dtype=torch.int64, device=cuda), inv)
    assert a.shape == b.shape == (2, 3, 0, 128)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Hq,Hkv,n,row,sections", [(1, 32, 8, 1, 0, None), (5, 14, 2, 1, 319, (16, 24, 24)), (64, 32, 8, 2, 100, None),
                                                     (2, 16, 11, 320, 0, (16, 24, 24))])
def test_step_write_is_norm_rotary_into_the_window(cuda, dtype, B, Hq, Hkv, n, row, sections):
    gen = torch.Generator(device=cuda).manual_seed(n + B)
    qkv = torch.randn(B, n, Hq + 2 * Hkv, 128, generator=gen, device=cuda).to(dtype)
    q, k, v = (x.transpose(1, 2) for x in qkv.split((Hq, Hkv, Hkv), dim=2))
    w = (1 + 0.3 * torch.randn(128, generator=gen, device=cuda)).to(dtype)
    pos = _pos(cuda, B, n, 9999, 3, gen)
    pos = pos if sections else pos[0]
    kw, vw = (torch.randn(B, Hkv, 320, 128, generator=gen, device=cuda).to(dtype) for _ in range(2))
    want_k, want_v = kw.clone(), vw.clone()
    wq, wk = ops.norm_rotary(q, k, pos, _inv(cuda), w, w, sections=sections)
    want_k[:, :, row:row + n], want_v[:, :, row:row + n] = wk, v
    gq = ops.window_append_rotary(q, k, v, pos, _inv(cuda), kw, vw, row, w, w, sections=sections)
    assert torch.equal(gq, wq) and torch.equal(kw, want_k) and torch.equal(vw, want_v)


def test_refusals(cuda):
    q, k = torch.zeros(2, 4, 3, 128, device=cuda).half(), torch.zeros(2, 2, 3, 128, device=cuda).half()
    pos, inv = torch.zeros(2, 3, dtype=torch.int64, device=cuda), _inv(cuda)
    win = torch.zeros(2, 2, 8, 128, device=cuda).half()

    def bad(match, fn=ops.norm_rotary, **kw):
        args = dict(q=q, k=k, positions=pos, inv_freq=inv)
        if fn is ops.window_append_rotary:
            args.update(v=k, k_win=win, v_win=win.clone(), win_pos=0)
        args.update(kw)
        with pytest.raises(RuntimeError, match=match):
            fn(**args)

    bad("one dtype", k=k.bfloat16())
    bad("Unsupported data type", q=q.float(), k=k.float())
    bad("one batch and length", k=k[:1])
    bad("one batch and length", k=k[..., :64])
    bad("int32 or int64", positions=pos.float())
    bad("broadcast", positions=pos[:, :2])
    bad("broadcast", positions=pos.expand(3, 2, 3))
    bad("broadcast", positions=pos.expand(2, 2, 3), sections=(16, 24, 24))
    bad("inv_freq", inv_freq=inv[:32])
    bad("norm weights", q_norm=torch.ones(128, device=cuda))
    bad("one device", positions=pos.cpu())
    bad("one device", k_norm=torch.ones(128).half())
    f = ops.window_append_rotary
    bad("do not fit", f, win_pos=6)
    bad("do not fit", f, win_pos=-1)
    bad("windows must", f, k_win=win[:, :, :, :64])
    bad("windows must", f, v_win=win.bfloat16())
    bad("K and V", f, v=k[:, :1])
    bad("one device", f, v=k.cpu())


def test_on_a_side_stream_and_in_a_graph(cuda):
    gen = torch.Generator(device=cuda).manual_seed(8)
    x = torch.randn(3, 1, 24, 128, generator=gen, device=cuda).half()
    q, k, v = (t.transpose(1, 2) for t in x.split((16, 4, 4), dim=2))
    pos, inv = torch.zeros(3, 1, dtype=torch.int64, device=cuda), _inv(cuda)
    kw, vw = (torch.zeros(3, 4, 64, 128, device=cuda).half() for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.window_append_rotary(q, k, v, pos, inv, kw, vw, 5)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.window_append_rotary(q, k, v, pos, inv, kw, vw, 5)
    for step in range(3):
        x.copy_(torch.randn(x.shape, generator=gen, device=cuda))
        pos.fill_(1000 * step + 3)
        graph.replay()
        wq, wk = ops.norm_rotary(q, k, pos, inv)
        torch.cuda.synchronize()
        assert torch.equal(out, wq) and torch.equal(kw[:, :, 5:6], wk) and torch.equal(vw[:, :, 5:6], v)


def test_no_heads_on_one_side_are_refused(cuda):
    q, pos, inv = torch.zeros(1, 4, 2, 128, device=cuda).half(), torch.arange(2, device=cuda), _inv(cuda)
    win = torch.zeros(1, 4, 8, 128, device=cuda).half()
    for a, b in ((q[:, :0], q), (q, q[:, :0])):
        with pytest.raises(RuntimeError, match="heads"):
            ops.norm_rotary(a, b, pos, inv)
    with pytest.raises(RuntimeError, match="heads"):
        ops.window_append_rotary(q[:, :0], q, q, pos, inv, win, win.clone(), 0)


def test_rows_further_apart_than_32_bits(cuda):
    """Inputs and a window whose second sequence and last heads start behind 2^31 elements."""
    gen = torch.Generator(device=cuda).manual_seed(9)
    flat = torch.empty((1 << 31) + 4096, dtype=torch.float16, device=cuda)
    q, k = flat.as_strided((2, 2, 3, 128), (1 << 31, 384, 128, 1)), flat.as_strided((2, 2, 3, 128), (1 << 31, 384, 128, 1), 1024)
    q.copy_(torch.randn(q.shape, generator=gen, device=cuda))
    k.copy_(torch.randn(k.shape, generator=gen, device=cuda))
    pos, inv = torch.arange(77, 80, device=cuda), _inv(cuda)
    want = ops.norm_rotary(q.contiguous(), k.contiguous(), pos, inv)
    got = ops.norm_rotary(q, k, pos, inv)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    cap = (1 << 22) + 70                                   # 2 x 2 x cap x 128 elements
    kw, vw = (torch.empty(2, 2, cap, 128, dtype=torch.float16, device=cuda) for _ in range(2))
    assert torch.equal(ops.window_append_rotary(q, k, q, pos, inv, kw, vw, cap - 3), want[0])
    assert torch.equal(kw[:, :, cap - 3:], want[1]) and torch.equal(vw[:, :, cap - 3:], q)
