"""The 8-bit operators' definitions in 64 bits on the CPU, and how far a kernel with fp32 sums may be from them."""
import torch

F8 = torch.float8_e4m3fn
TOP, LEAST = 448.0, 2.0 ** -100
U = 2.0 ** -24                            # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step among the smallest numbers of the type."""
    return torch.finfo(dtype).smallest_normal * half_step(dtype)


def scales(y, block):
    """Scales of y [rows, width] in 64 bits, of finite values alone."""
    rows, width = y.shape
    size = torch.where(torch.isfinite(y), y.abs(), torch.zeros_like(y))
    size = torch.nn.functional.pad(size, (0, -width % 128, 0, -rows % block))
    return size.view(-1, block, size.size(1) // 128, 128).amax(dim=(1, 3)).clamp_min(LEAST) / TOP


def spread(scale, block, rows, width):
    return scale.double().repeat_interleave(block, 0)[:rows].repeat_interleave(128, 1)[:, :width]


def check_eight(e, y, block, rel=0.0):
    """Codes and scales `e` of the values y [rows, width] (64 bits; the kernel's own may be off by `rel` of them)."""
    codes, scale = e["codes"].cpu().reshape(y.shape), e["scale"].cpu().reshape(-1, e["scale"].size(-1)).double()
    want = scales(y, block)
    assert scale.shape == want.shape
    assert bool(((scale - want).abs() <= (rel + 2 * U) * want).all()), ((scale - want).abs() / want).max().item()
    q = y / spread(want, block, *y.shape)
    c = codes.double()
    fine = torch.isfinite(y)
    assert bool(torch.isnan(c[~fine]).all())
    c, q = c[fine], q[fine]
    size = torch.maximum(c.abs(), q.abs())
    step = torch.exp2(torch.floor(torch.log2(size.clamp_min(2.0 ** -6))) - 3)          # of e4m3 at this size; 2^-9 among its smallest
    # value and scale off by rel, the scale's and the quotient's three roundings
    err = (c - q).abs() - (0.5 * step + (2 * rel + 4 * U) * q.abs())
    assert bool((err <= 0).all()), (err.max().item(), c[err.argmax()].item(), q[err.argmax()].item())


def make_eight(y, block):
    """The 8-bit form of y [rows, width], 32 bits, by elementary operations (for inputs)."""
    s = scales(y.double(), block).float()
    return {"codes": (y / spread(s, block, *y.shape).float()).to(F8), "scale": s}


def product(x, w, block=128):
    """(sum, tolerance before the last rounding, its mean square) of x [M, K] times w [N, K] transposed, 8-bit forms (a scale of w for
    `block` rows).

    The instruction's sums: every product is cut by less than 2^-13 of the power of two of its group of eight's largest, groups are added in
    fp32, 16 of them, each addition off by a step at most (2 U) of what is added up; a block's sum gets its scales (their product rounded once)
    and is added to a chain of as many as there are blocks, and eight wavefronts' chains are joined, one rounding each."""
    xc, wc = x["codes"].cpu().double(), w["codes"].cpu().double()
    M, K = xc.shape
    N, blocks = wc.size(0), -(-K // 128)
    xs, ws = x["scale"].cpu().double().reshape(M, blocks), w["scale"].cpu().double().repeat_interleave(block, 0)[:N]
    y, tol, var = (torch.zeros(M, N, dtype=torch.float64) for _ in range(3))
    for b in range(blocks):
        xa, wa = (torch.nn.functional.pad(c[:, 128 * b:128 * b + 128], (0, -min(K - 128 * b, 128) % 8)) for c in (xc, wc))
        f = xs[:, b, None] * ws[None, :, b]
        y += (xa @ wa.t()) * f
        mass = (xa.abs() @ wa.abs().t()) * f
        tol += mass * U * (32 + blocks + 10)
        for k in range(0, xa.size(1), 8):
            top = (xa[:, None, k:k + 8].abs() * wa[None, :, k:k + 8].abs()).amax(-1) * f
            tol += 8 * 2.0 ** -13 * top
            var += 8 * (2.0 ** -13 * top) ** 2
    return y, tol, var


def check_rounded(got, want, tol, var):
    """16-bit results against 64 bits: each within its tolerance and half a step; together within what independent cuts and the rounding give."""
    got = got.cpu().reshape(want.shape)
    h = half_step(got.dtype)
    over = want.abs() > torch.finfo(got.dtype).max
    assert not bool(over.any())
    err = (got.double() - want).abs()
    allowed = tol + h * (want.abs() + tol) + tiny(got.dtype)
    assert bool((err <= allowed).all()), (err.max().item(), (err / allowed).max().item())
    rms = lambda t: float(t.square().mean().sqrt())
    assert rms(err) <= h * rms(want) + 2 * float(var.mean().sqrt()) + tiny(got.dtype), (rms(err), rms(want))


def gated(g, u):
    """(result, tolerance, mean square) of silu(g) u from product()'s for both.  silu's slope is below 1.1; exp takes |g| + 4 roundings (its
    argument is scaled in fp32), sum, quotient and product four more."""
    (yg, tg, vg), (yu, tu, vu) = g, u
    s = yg * torch.sigmoid(yg)
    y = s * yu
    tol = 1.1 * tg * (yu.abs() + tu) + s.abs() * tu + y.abs() * U * 2 * (yg.abs() + 8)
    return y, tol, (1.1 * yu) ** 2 * vg + s ** 2 * vu
