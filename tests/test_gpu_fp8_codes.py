"""Codes of the 8-bit form bit for bit: the fp32 quotient of value and scale, rounded to the nearest e4m3, ties to even.

The kernels form it as q = y * inv, q + (y - q * s) * inv, inv = 1 / s to a step (2^-23).  q is off by 3 * 2^-23 at most, the remainder (26 bits) loses 2^-24 of
itself: before the last rounding the sum is y / s to 2^-43.  Where that rounds as the division does, the codes are the same; where it does not, they
can differ only if y / s is within a step of the middle m of two codes (five bits).  For 16-bit values y, and M the block's largest, that never happens:
s = M / 448 (1 + e), |e| <= 2^-24, so y / s = 448 y / M / (1 + e), and 448 y - m M, of numbers of 14 and 16 bits, is zero or 2^-16 of them.  Zero with e = 0: y / s = m, and
the sum is m, too.  Zero with e != 0: seven does not divide M, so it divides m, m = 21 / 16 times a power of two, and the division gives m where
|e| < 2^-24 * 16 / 21 and a neighbour otherwise; the sum could differ only if |e| were that to 2^-19 of itself.  M / 7 is off a step of s by n / 7 steps,
|e| = n / (7 f) 2^-23, n = 1, 2 or 3, f in [1, 2) the significand of s: it would take f = 3 n / 8 = 9 / 8 to 2^-19, which M = 63 * 2^i has (a multiple of seven) and no other
eleven bits come that near to."""
import pytest
import torch

import fp8_oracle as oracle
from packkv_amd import ops

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def _divided(x, scale, block):
    """codes of x [rows, width] by an fp32 division on the CPU"""
    s = scale.repeat_interleave(block, 0)[:x.size(0)].repeat_interleave(128, 1)[:, :x.size(1)]
    return (x.float() / s).to(oracle.F8).view(torch.uint8)


def _rows(dtype):
    """Every significand as a block's largest value, and beside it the values at and next to the middles of two codes."""
    digits = 11 if dtype == torch.float16 else 8
    top = torch.arange(1 << digits - 1, 1 << digits).double()[:, None]
    odd = torch.arange(17, 32, 2).double()
    middles = torch.cat([odd[:6] / 28] + [odd / 28 / 2 ** i for i in range(1, 6)])[None]     # over the largest value, which is the code 448 = 28 * 16
    step = torch.exp2(torch.floor(torch.log2(top * middles)) - (digits - 1))
    at = (top * middles / step).round()
    near = torch.cat(((at + 1) * step, at * step, (at - 1) * step), dim=1)[:, :127]
    return torch.cat((top, torch.minimum(near, top)), dim=1).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_codes_are_the_quotients(cuda, dtype):
    x = _rows(dtype)
    assert x.size(1) == 128
    e = ops.fp8_quantize(x.to(cuda))
    scale = e["scale"].cpu()
    assert torch.equal(scale, x.float().amax(1, keepdim=True) / 448)
    assert torch.equal(e["codes"].cpu().view(torch.uint8), _divided(x, scale, 1))
    # the same as weights, a row's values in a block of their own
    b = torch.zeros(4 * 128, 16 * 128, dtype=dtype)
    some = x[torch.linspace(0, x.size(0) - 1, 64).long()]
    b[::128] = some.view(4, 16 * 128)
    e = ops.fp8_quantize(b.to(cuda), 128)
    assert torch.equal(e["codes"].cpu().view(torch.uint8), _divided(b, e["scale"].cpu(), 128))


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_codes_of_values_that_fp32_holds(cuda, dtype):
    """Rows of one size, 64 and -64, have a norm of exactly their signs (eps 0); the weight's values are what is quantized then."""
    w = _rows(dtype)
    w = w[torch.linspace(0, w.size(0) - 1, 32).long()].reshape(-1)
    sign = torch.where(torch.rand(5, w.numel(), generator=torch.Generator().manual_seed(0)) < 0.5, -1.0, 1.0)
    e = ops.add_rms_norm((64 * sign).to(dtype).to(cuda), w.to(cuda), 0.0, fp8=True)
    y = (sign * w.float()).view(-1, 128)
    scale = e["scale"].cpu().reshape(-1, 1)
    assert torch.equal(scale, y.abs().amax(1, keepdim=True) / 448)
    assert torch.equal(e["codes"].cpu().view(-1, 128).view(torch.uint8), _divided(y, scale, 1))


@pytest.mark.parametrize("dtype", TYPES)
def test_codes_of_ordinary_values_are_the_quotients(cuda, dtype):
    gen = torch.Generator().manual_seed(3)
    x = (torch.randn(3000, 912, generator=gen) * torch.exp(torch.randn(3000, 1, generator=gen))).to(dtype)
    x[:, ::7] *= 0                                         # zeroes of both signs
    for block in (1, 128):
        e = ops.fp8_quantize(x.to(cuda), block)
        assert torch.equal(e["codes"].cpu().view(torch.uint8), _divided(x, e["scale"].cpu(), block))
