"""attn_chunk with codes wider than 4 bits on one side or both, in every form of the call: windows, left padding, without the causal
mask, both types, from a few rows to many; and the same call again, bit for bit."""
import pytest
import torch

import chunk_oracle as co
from chunk_drawn import drawn
from packkv_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k_bits,v_bits", [(5, 5), (5, 4), (4, 5), (6, 6), (4, 8), (8, 3), (8, 8), (4, 4)])
@pytest.mark.parametrize("n", [3, 12, 40])                 # with four query heads to a KV head: up to 32 rows, up to 64, more
def test_every_form(cuda, dtype, k_bits, v_bits, n):
    B, H, G, T, W = 2, 2, 4, 512, 77
    print("wide case", dtype, k_bits, v_bits, n, flush=True)
    g = torch.Generator(device=cuda).manual_seed(k_bits * 16 + v_bits + n)
    k, v = drawn(cuda, True, B, H, T, k_bits, dtype, g), drawn(cuda, False, B, H, T, v_bits, dtype, g)
    kw, vw = (torch.randn(B, H, 100, 128, generator=g, device=cuda).to(dtype) for _ in range(2))
    q = torch.randn(B, n, G * H, 128, generator=g, device=cuda).to(dtype).transpose(1, 2)
    K, sizes = co.values_of(k, True, B, H, kw, W)
    V, v_sizes = co.values_of(v, False, B, H, vw, W)
    size = dict(sizes=sizes, v_sizes=v_sizes)
    co.check(ops.attn_chunk(q, k, v, kw, vw, win_len=W), q, K, V, **size)
    co.check(ops.attn_chunk(q, k, v, kw, vw, win_len=W, causal=False, sm_scale=0.05), q, K, V, causal=False, sm=0.05, **size)
    bare = dict(sizes=sizes[:, :, :T], v_sizes=v_sizes[:, :, :T])
    co.check(ops.attn_chunk(q, k, v), q, K[:, :, :T], V[:, :, :T], **bare)
    for starts in ((130, T + 5), (T + W - 2, T - 1)):
        st = torch.tensor(starts, dtype=torch.int32, device=cuda)
        got = ops.attn_chunk(q, k, v, kw, vw, win_len=W, starts=st)
        co.check(got, q, K, V, starts=list(starts), **size)
        for b, s in enumerate(starts):
            assert bool((got[b, :, :max(0, min(n, s - (T + W - n)))] == 0).all())


@pytest.mark.parametrize("dtype,bits", [(torch.float16, 4), (torch.bfloat16, 4), (torch.bfloat16, 5)])
@pytest.mark.parametrize("B,n,T", [(1, 3, 896), (4, 4, 8192), (2, 333, 2048)])
def test_the_same_call_gives_the_same_bits(cuda, dtype, bits, B, n, T):
    H, G, W = 2, 4, 50
    g = torch.Generator(device=cuda).manual_seed(n)
    k, v = drawn(cuda, True, B, H, T, bits, dtype, g), drawn(cuda, False, B, H, T, bits, dtype, g)
    kw, vw = (torch.randn(B, H, W, 128, generator=g, device=cuda).to(dtype) for _ in range(2))
    q = torch.randn(B, n, G * H, 128, generator=g, device=cuda).to(dtype).transpose(1, 2)
    first = ops.attn_chunk(q, k, v, kw, vw)
    for _ in range(5):
        ops.attn_chunk(q.flip(2), k, v, kw, vw)
        assert torch.equal(ops.attn_chunk(q, k, v, kw, vw), first)
