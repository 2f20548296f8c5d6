"""attn_chunk with queries of far-apart sizes: a row's scores come from its own query, however large the other rows' are."""
import pytest
import torch

from chunk_drawn import check, drawn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 5])
@pytest.mark.parametrize("G,n,W", [(4, 3, 0), (4, 4, 20), (4, 7, 0), (4, 12, 9), (4, 40, 0), (1, 200, 0)])
@pytest.mark.parametrize("apart", [12, 40, 100])
def test_rows_of_far_apart_sizes(cuda, bits, G, n, W, apart):
    """bf16 queries about 2^-apart beside one of usual size and a row of zeroes, keys about 2^apart: the small rows' scores are of the
    usual size, the large row's attention is a peak."""
    B, H, T, dtype = 2, 2, 384, torch.bfloat16
    g = torch.Generator(device=cuda).manual_seed(n + apart)
    k, v = drawn(cuda, True, B, H, T, bits, dtype, g), drawn(cuda, False, B, H, T, bits, dtype, g)
    k["scale"] *= 2.0 ** apart
    kw, vw = ((torch.randn(B, H, W, 128, generator=g, device=cuda) * s).to(dtype) if W else None for s in (2.0 ** apart, 1.0))
    q = (torch.randn(B, n, G * H, 128, generator=g, device=cuda) * 2.0 ** -apart).to(dtype).transpose(1, 2)
    q[:, G * H - 1, n // 2] *= 2.0 ** apart
    q[1, 0, n - 1] = 0
    check(q, k, v, kw, vw, W)
