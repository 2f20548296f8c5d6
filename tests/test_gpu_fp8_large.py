"""Products with weights past 4 GiB, through the kernels for few rows and for many: results whose rows of weights lie on either side of it."""
import pytest
import torch

import fp8_oracle as oracle
from packkv_amd import ops

pytestmark = pytest.mark.gpu
ROWS, WIDTH = (1 << 20) + 4000, 4112


@pytest.fixture(scope="module")
def weights(cuda):
    """Zeroes but for some gate rows n, at the 4 GiB of their up rows n + ROWS / 2 and elsewhere, and those up rows."""
    assert ROWS * WIDTH > 1 << 32
    gen = torch.Generator(device=cuda).manual_seed(5)
    n, edge = ROWS // 2, (1 << 32) // WIDTH
    at = torch.tensor([0, 5, edge - n - 1, edge - n, edge - n + 1, edge - n + 2, n - 17, n - 1], device=cuda)
    codes = torch.zeros(ROWS, WIDTH, dtype=torch.uint8, device=cuda)
    some = torch.randint(-2, 3, (2 * at.numel(), WIDTH), generator=gen, device=cuda).float().to(oracle.F8)
    codes[torch.cat((at, at + n))] = some.view(torch.uint8)
    yield {"codes": codes.view(oracle.F8), "scale": torch.full((-(-ROWS // 128), -(-WIDTH // 128)), 2.0 ** -6, device=cuda)}, at, some.double() / 64


@pytest.mark.parametrize("rows", [1, 40, 128, 256])
def test_linear_and_gated(cuda, weights, rows):
    w, at, some = weights
    codes = torch.randint(-2, 3, (rows, WIDTH), generator=torch.Generator(device=cuda).manual_seed(rows), device=cuda).float().to(oracle.F8)
    x = {"codes": codes, "scale": torch.ones(rows, -(-WIDTH // 128), device=cuda)}
    y = codes.double() @ some.t().contiguous()               # (exact in fp32 too: whole numbers over 64)
    got = ops.fp8_linear(x, w)
    both = torch.cat((at, at + ROWS // 2))
    assert torch.equal(got[:, both], y.bfloat16())
    got[:, both] = 0
    assert not bool(got.any())
    del got
    g, u = y.chunk(2, dim=1)
    want = g * torch.sigmoid(g) * u
    assert bool((want != 0).any(dim=0).all())
    got = ops.fp8_gated(x, w)
    # the last rounding; exp's argument and the three operations behind it (fp8_oracle.gated)
    tol = (oracle.half_step(torch.bfloat16) + 2 * oracle.U * (g.abs() + 8)) * want.abs() + oracle.tiny(torch.bfloat16)
    assert bool(((got[:, at].double() - want).abs() <= tol).all())
    got[:, at] = 0
    assert not bool(got.any())


@pytest.mark.parametrize("gated", [False, True])
def test_results_beyond_4_gib(cuda, gated):
    gen = torch.Generator(device=cuda).manual_seed(1)
    rows, cols = 2113, ROWS
    draw = lambda n: torch.randint(-2, 3, (n, 16), generator=gen, device=cuda).float()
    x, w = draw(rows), draw((2 if gated else 1) * cols)
    assert 2 * rows * cols > 1 << 32
    eight = lambda t, block: {"codes": t.to(oracle.F8), "scale": torch.full((-(-t.size(0) // block), 1), 0.25, device=cuda)}
    got = (ops.fp8_gated if gated else ops.fp8_linear)(eight(x, 1), eight(w, 128))
    assert got.shape == (rows, cols)
    for m in (slice(0, 70), slice(1000, 1070), slice((1 << 31) // cols - 2, (1 << 31) // cols + 3), slice(rows - 70, rows)):
        y = (x[m] @ w.t().contiguous()) / 16                 # (exact)
        if not gated:
            assert torch.equal(got[m], y.bfloat16())
            continue
        g, u = y[:, :cols].double(), y[:, cols:].double()
        want = g * torch.sigmoid(g) * u
        tol = (oracle.half_step(torch.bfloat16) + 2 * oracle.U * (g.abs() + 8)) * want.abs() + oracle.tiny(torch.bfloat16)
        assert bool(((got[m].double() - want).abs() <= tol).all())
