"""attn_chunk where sizes lie far apart: a row's result comes from its own query and from the tokens it sees, whatever finite numbers
the other rows and the later tokens hold.  Against attention in 64 bits (chunk_oracle), whose tolerance is relative to the row's own."""
import pytest
import torch

from chunk_drawn import check, drawn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [4, 5])
@pytest.mark.parametrize("G,n", [(4, 4), (1, 16), (4, 7), (4, 12), (4, 31), (2, 130), (1, 300)])
@pytest.mark.parametrize("shape", ["rising", "jump", "jumps"])
def test_later_tokens_scales_do_not_reach_a_row(cuda, dtype, bits, G, n, shape):
    """V scales that rise inside the new tokens: from token to token, or at one or several of them, by up to 2^24 (bf16: 2^56)."""
    B, H, T = 2, 2, 512
    g = torch.Generator(device=cuda).manual_seed(n + G + bits)
    k, v = drawn(cuda, True, B, H, T, bits, dtype, g), drawn(cuda, False, B, H, T, bits, dtype, g)
    top = 24 if dtype == torch.float16 else 56
    at = torch.arange(T, device=cuda) - (T - n)
    if shape == "rising":
        up = at.clamp_min(0) * max(1, -(-top // n))
    elif shape == "jump":
        up = torch.where(at == n - 1, top, 0)
    else:
        up = (at.clamp_min(0) * 4 // n) * (top // 3)
    scale = 2.0 ** (up.clamp_max(top).double() - 14)
    v["scale"] = (scale * (1.0 + 0.5 * torch.rand(B, T, generator=g, device=cuda).double())).to(dtype)
    assert bool(v["scale"].isfinite().all()) and v["scale"].min().item() >= 2.0 ** -14
    q = torch.randn(B, n, G * H, 128, generator=g, device=cuda).to(dtype).transpose(1, 2)
    check(q, k, v)
    check(q, k, v, starts=torch.tensor([3, T - n + n // 3], dtype=torch.int32, device=cuda))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("G,n,W", [(4, 9, 4), (2, 70, 33), (4, 4, 2)])
def test_later_tokens_scales_with_a_window_behind(cuda, dtype, G, n, W):
    """The same where the last of the new tokens are in the window, whose values are of the rows' usual size."""
    B, H, T = 1, 2, 256
    g = torch.Generator(device=cuda).manual_seed(n + W)
    k, v = drawn(cuda, True, B, H, T, 4, dtype, g), drawn(cuda, False, B, H, T, 4, dtype, g)
    first = T - (n - W)                                    # the first new token; only rows behind it see what it holds
    v["scale"][:, :first] *= 2.0 ** -8
    v["scale"][:, first + 2:] *= 2.0 ** (14 if dtype == torch.float16 else 40)
    kw, vw = (torch.randn(B, H, W, 128, generator=g, device=cuda).to(dtype) for _ in range(2))
    q = torch.randn(B, n, G * H, 128, generator=g, device=cuda).to(dtype).transpose(1, 2)
    check(q, k, v, kw, vw, W)
