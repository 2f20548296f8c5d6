"""fp8_gated at the ends of fp32's range: whatever silu(gate) * up is in bf16, with gates and ups that fp32 holds.

One code of 1 in x and scales that are powers of two make every gate and every up a code times a power of two, exact in fp32 with no product
cut; the rest of the tolerance is the operator's own: exp's |g| + 4 roundings and sum, quotient, product (fp8_oracle.gated), and the last one."""
import pytest
import torch

import fp8_oracle as oracle
from packkv_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 40, 700, 4000])
@pytest.mark.parametrize("gate,up", [(124, -124), (124, -3), (124, 0), (119, -119), (62, 60), (0, 120), (0, -60), (-60, 60), (-120, 120), (-110, 0)])
def test_gated_where_fp32_ends(cuda, rows, gate, up):
    """Gates of code * 2^gate, up to 15 * 2^124 (fp32 ends at 2^128), against ups of code * 2^up, zero among them."""
    codes = torch.tensor([0.0, 1, -1, 1.5, 7, -7, 15, -15, 2.0 ** -9, 0.875, 80, -80, 88, -88, 0.0625, -0.0625])
    n = codes.numel()
    gates, ups = codes[(codes.abs() <= 15) | (torch.tensor(gate) < 100)].repeat(2)[:n], codes.clamp(-15, 15)
    pairs = torch.cartesian_prod(torch.arange(n), torch.arange(n))[torch.randperm(n * n, generator=torch.Generator().manual_seed(rows))[:128]]
    g, u = gates[pairs[:, 0]], ups[pairs[:, 1]]
    xc, wc = torch.zeros(rows, 128), torch.zeros(256, 128)
    xc[:, 0] = 1
    wc[:128, 0], wc[128:, 0] = g, u
    x = {"codes": xc.to(oracle.F8).to(cuda), "scale": torch.full((rows, 1), 1.0, device=cuda)}
    w = {"codes": wc.to(oracle.F8).to(cuda), "scale": torch.tensor([[2.0 ** gate], [2.0 ** up]], device=cuda)}
    assert torch.equal(w["codes"].float().cpu(), wc)
    got = ops.fp8_gated(x, w).cpu()
    gd, ud = g.double() * 2.0 ** gate, u.double() * 2.0 ** up
    want = gd * torch.sigmoid(gd) * ud
    assert bool(torch.isfinite(got[:, want.abs() < 2.0 ** 127]).all())
    # (e^-g of fp32 is infinite from -88.7 on; up's quarter is a multiple of 2^-149, off by 2^-150, and four times that comes with at most g;
    # its product with the reciprocal is off by 2^-150 once more, times g; bf16 has eight significant bits: half a step is 2^-8 of a value)
    fine = (want.abs() < 2.0 ** 127) & (gd > -88.5)
    tol = (oracle.half_step(torch.bfloat16) + 2 * oracle.U * (gd.abs().clamp_max(90) + 8)) * want.abs() + oracle.tiny(torch.bfloat16) + 2.0 ** -147 * gd.abs()
    err = (got.double() - want).abs() - tol
    assert bool((err[:, fine] <= 0).all()), (err[:, fine].max().item(), gd[fine], ud[fine], got[0, fine])
    assert bool((got[:, ud == 0] == 0).all())


@pytest.mark.parametrize("rows", [1, 40, 700])
@pytest.mark.parametrize("xs,ws", [(-60, -60), (-60, -75), (-109, -30), (-100, -100), (60, -109), (100, -140)])
def test_linear_of_small_scales(cuda, rows, xs, ws):
    """The product of a block's two scales is an fp32 number: below 2^-126 a multiple of 2^-149, off by 2^-150 at most.  (Whole codes -2 .. 2 and no cut: the
    rest is a rounding for the scales' product, one a block, and the last one.)"""
    gen = torch.Generator().manual_seed(rows)
    width, cols = 400, 272
    whole = lambda *shape: torch.randint(-2, 3, shape, generator=gen).float()
    draw = lambda blocks, e: ((1 + torch.rand(blocks, 4, generator=gen)) * 2.0 ** e).to(cuda)
    x, w = {"codes": whole(rows, width).to(oracle.F8).to(cuda), "scale": draw(rows, xs)}, {"codes": whole(cols, width).to(oracle.F8).to(cuda), "scale": draw(3, ws)}
    y, mass, sums = (torch.zeros(rows, cols, dtype=torch.float64) for _ in range(3))
    for b in range(4):
        xa, wa = (t["codes"].cpu().double()[:, 128 * b:128 * b + 128] for t in (x, w))
        f = x["scale"].cpu().double()[:, b, None] * w["scale"].cpu().double().repeat_interleave(128, 0)[:cols, b][None]
        d = xa @ wa.t()
        y, mass, sums = y + d * f, mass + d.abs() * f, sums + d.abs()
    got = ops.fp8_linear(x, w).cpu().double()
    tol = 12 * oracle.U * mass + 2.0 ** -150 * (sums + 12)
    err = (got - y).abs()
    assert bool((err <= tol + oracle.half_step(torch.bfloat16) * (y.abs() + tol) + oracle.tiny(torch.bfloat16)).all())
