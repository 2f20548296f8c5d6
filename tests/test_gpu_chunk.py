"""attn_chunk -- several new tokens over a compressed cache -- against attention in 64 bits on the codes, parameters and window."""
import pytest
import torch

import chunk_oracle as co
from packkv_amd import _lib, ops, synth
from packkv_amd.cache import PackKVCacheConfig, PackKVCompressedCache

pytestmark = pytest.mark.gpu


def _case(cuda, B, Hq, Hkv, n, T, W, dtype, k_rel=0.1, v_rel=0.1, seed=0, cap=320):
    k, v = synth.make_kv(B, Hkv, T + cap, seed=seed, dtype=dtype, device=cuda)
    ke = ve = kw = vw = None
    if T:
        ke, ve = ops.k_quant_encode(k[:, :, :T].contiguous(), k_rel), ops.v_quant_encode(v[:, :, :T].contiguous(), v_rel)
        ke["heads"] = ve["heads"] = Hkv
    if W:
        kw, vw = k[:, :, T:].contiguous(), v[:, :, T:].contiguous()
    g = torch.Generator(device=cuda).manual_seed(seed + 1)
    q = torch.randn(B, n, Hq, 128, generator=g, device=cuda).to(dtype).transpose(1, 2)
    return q, ke, ve, kw, vw


def _values(ke, ve, kw, vw, B, H, W):
    K, sizes = co.values_of(ke, True, B, H, kw, W)
    V, v_sizes = co.values_of(ve, False, B, H, vw, W)
    return K, V, dict(sizes=sizes, v_sizes=v_sizes)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Hq,Hkv,n,T,W", [
    (1, 1, 1, 1, 128, 0), (1, 8, 1, 2, 128, 1), (2, 32, 8, 3, 896, 201), (1, 4, 4, 32, 256, 31), (3, 14, 2, 5, 1024, 255), (1, 40, 8, 33, 384, 129),
    (2, 8, 2, 130, 128, 3), (1, 16, 1, 77, 640, 320), (1, 2, 2, 7, 0, 7), (2, 4, 1, 60, 0, 300), (1, 32, 8, 300, 4096, 64), (1, 10, 1, 128, 128, 0),
    (9, 8, 8, 1, 2048, 5), (1, 8, 2, 4, 33024, 100)])
def test_chunk_follows_the_formula(cuda, dtype, B, Hq, Hkv, n, T, W):
    print("chunk case", B, Hq, Hkv, n, T, W, dtype, flush=True)
    q, ke, ve, kw, vw = _case(cuda, B, Hq, Hkv, n, T, W, dtype, seed=n + T)
    K, V, size = _values(ke, ve, kw, vw, B, Hkv, W)
    got = ops.attn_chunk(q, ke, ve, kw, vw, win_len=W or None)
    assert got.shape == q.shape and got.dtype == dtype and got.stride() == torch.empty_like(q).stride()
    co.check(got, q, K, V, **size)


@pytest.mark.parametrize("k_bits,v_bits", [(2, 2), (3, 4), (4, 3), (5, 4), (4, 6), (6, 5), (8, 7), (7, 8), (5, 5), (6, 6), (8, 8), (8, 2), (2, 8)])
@pytest.mark.parametrize("B,Hq,Hkv,n,T", [(2, 8, 2, 17, 384), (2, 32, 8, 40, 4096), (4, 8, 8, 3, 8192)])
def test_every_width(cuda, k_bits, v_bits, B, Hq, Hkv, n, T):
    """Codes that use their whole width (drawn, not quantised), with packs of every length; one tile a workgroup, and runs of several
    with many rows and with few (the staged blocks of wide codes then lie beyond 64 KiB of LDS)."""
    dtype = torch.float16
    g = torch.Generator(device=cuda).manual_seed(k_bits * 10 + v_bits)
    sides = []
    for is_k, bits in ((True, k_bits), (False, v_bits)):
        span = torch.randint(1, (1 << bits) + 1, (T // 16, 1, B * Hkv * 128), generator=g, device=cuda)
        codes = (torch.rand(T // 16, 16, B * Hkv * 128, generator=g, device=cuda) * span).long().clamp_(max=(1 << bits) - 1)
        codes = codes.to(torch.uint8).view(T, -1)
        blocks = (T // (64 if is_k else 128)) * (B * Hkv * (1 if is_k else 2))
        stream = torch.empty(blocks * ops.block_bound(is_k, 64 if is_k else 128, 128 if is_k else 64, bits) + 16, dtype=torch.uint8, device=cuda)
        info = torch.empty(blocks, 2, dtype=torch.uint32, device=cuda)
        size = (ops.k_encode if is_k else ops.v_encode)(codes, stream, info, bits=bits)
        scale = ((0.5 + torch.rand(B, T, generator=g, device=cuda)) * 2.0 / (1 << bits)).to(dtype)
        zero = (-(1 << bits) * torch.rand(B, T, generator=g, device=cuda)).to(dtype)
        sides.append({"stream": stream[:size].clone(), "info": info, "scale": scale, "zero": zero, "bits": bits, "size": size, "heads": Hkv})
    q = torch.randn(B, Hq, n, 128, generator=g, device=cuda).to(dtype)
    K, V, size = _values(sides[0], sides[1], None, None, B, Hkv, 0)
    co.check(ops.attn_chunk(q, sides[0], sides[1]), q, K, V, **size)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,T,W,starts", [(5, 512, 40, (0, 551, 552, 300)), (300, 256, 100, (128, 127, 256, 356)), (40, 0, 90, (89, 90, 1000, 50)),
                                          (64, 384, 0, (-5, 383, 320, 384)), (3, 512, 40, (0, 551, 552, 300)), (4, 256, 0, (255, 256, 100, 3)),
                                          (2, 0, 170, (169, 170, 33, 1)), (1, 256, 129, (384, 385, 256, 0)), (8, 256, 20, (270, 275, 276, 31))])
def test_padding_on_the_left(cuda, dtype, n, T, W, starts):
    """Starts in streams and window, on and off tile borders, rows that see one token and rows that see none; what lies in the
    padding is NaN or infinite."""
    B, Hq, Hkv = 4, 8, 2
    q, ke, ve, kw, vw = _case(cuda, B, Hq, Hkv, n, T, W, dtype, seed=5)
    K, V, size = _values(ke, ve, kw, vw, B, Hkv, W)
    st = torch.tensor(starts, dtype=torch.int32, device=cuda)
    want = dict(starts=[min(max(s, 0), T + W) for s in starts], **size)
    co.check(ops.attn_chunk(q, ke, ve, kw, vw, win_len=W or None, starts=st), q, K, V, **want)
    for b, s in enumerate(starts):
        for i, side in enumerate((ke, ve)):
            if side is not None:
                side["scale"][b, :max(s, 0)] = float("inf")
                side["zero"][b, :max(s, 0)] = float("nan")
        if W and s > T:
            kw[b, :, :s - T], vw[b, :, :s - T] = float("nan"), float("inf")
    got = ops.attn_chunk(q, ke, ve, kw, vw, win_len=W or None, starts=st)
    co.check(got, q, K, V, **want)
    for b, s in enumerate(starts):
        blind = max(0, min(n, s - (T + W - n)))
        assert bool((got[b, :, :blind] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,W", [(9, 40), (60, 61), (6, 70)])
def test_queries_in_the_padding_and_broken_ones(cuda, dtype, n, W):
    """Queries of padded places, and those of one head that are infinite or NaN, leave every other row as it was."""
    B, Hq, Hkv, T = 2, 8, 4 if n < 9 else 2, 256
    q, ke, ve, kw, vw = _case(cuda, B, Hq, Hkv, n, T, W, dtype, seed=9)
    st = torch.tensor([T + W - n + 4, 0], dtype=torch.int32, device=cuda)
    want = ops.attn_chunk(q, ke, ve, kw, vw, win_len=W, starts=st)
    assert bool((want[0, :, :4] == 0).all()) and bool(want[0, :, 4:].any())
    big = torch.finfo(dtype).max
    q[0, 0, :4], q[0, 1, :4], q[0, 2:, :4] = float("nan"), float("inf"), big
    assert torch.equal(ops.attn_chunk(q, ke, ve, kw, vw, win_len=W, starts=st), want)
    q[1, 3, 2, 5], q[1, 3, 5, 7] = float("inf"), float("nan")
    got = ops.attn_chunk(q, ke, ve, kw, vw, win_len=W, starts=st)
    q[1, 3, 2, 5] = q[1, 3, 5, 7] = 0
    others = torch.ones(q.shape[:3], dtype=torch.bool, device=cuda)
    others[1, 3, 2] = others[1, 3, 5] = False
    assert torch.equal(got[others], want[others]) and bool(got[1, 3, 5].isnan().all())


def test_rows_behind_the_last_token_are_not_read(cuda):
    q, ke, ve, kw, vw = _case(cuda, 2, 8, 2, 6, 256, 70, torch.bfloat16)
    want = ops.attn_chunk(q, ke, ve, kw, vw, win_len=70)
    kw[:, :, 70:], vw[:, :, 70:] = float("nan"), float("inf")
    assert torch.equal(ops.attn_chunk(q, ke, ve, kw, vw, win_len=70), want)


def test_without_the_causal_mask_and_with_a_scale(cuda):
    B, Hq, Hkv, n, T, W = 2, 12, 4, 9, 256, 33
    q, ke, ve, kw, vw = _case(cuda, B, Hq, Hkv, n, T, W, torch.float16)
    K, V, size = _values(ke, ve, kw, vw, B, Hkv, W)
    co.check(ops.attn_chunk(q, ke, ve, kw, vw, win_len=W, causal=False, sm_scale=0.3), q, K, V, causal=False, sm=0.3, **size)
    many = q.repeat(1, 1, 40, 1)                           # more queries than tokens
    co.check(ops.attn_chunk(many, ke, ve, kw, vw, win_len=W, causal=False), many, K, V, causal=False, **size)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_and_queries_of_far_apart_sizes(cuda, dtype):
    """Token scales over many powers of two, growing and falling; one head's queries tiny beside another's; a peaked row."""
    B, Hq, Hkv, n, T, W = 1, 8, 2, 20, 1024, 50
    q, ke, ve, kw, vw = _case(cuda, B, Hq, Hkv, n, T, W, dtype)
    span = 2.0 ** torch.linspace(-9, 9, T, device=cuda)
    for perm in (torch.arange(T, device=cuda), torch.arange(T, device=cuda).flip(0)):
        ve2 = dict(ve, scale=(ve["scale"].float() * span[perm]).to(dtype))
        q2 = q.clone()
        q2[:, 0] *= 2.0 ** -12
        q2[:, 1] *= 6
        K, V, size = _values(ke, ve2, kw, vw, B, Hkv, W)
        co.check(ops.attn_chunk(q2, ke, ve2, kw, vw, win_len=W), q2, K, V, **size)


def test_layouts_of_queries_and_results(cuda):
    q, ke, ve, kw, vw = _case(cuda, 2, 8, 2, 6, 256, 70, torch.float16)
    want = ops.attn_chunk(q.contiguous(), ke, ve, kw, vw, win_len=70)
    flat = torch.zeros(2 * 8 * 6 * 131 + 1, device=cuda).half()
    odd = flat[1:].as_strided(q.shape, (8 * 6 * 131, 6 * 131, 131, 1))
    odd.copy_(q)
    for same in (q, odd, q.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(ops.attn_chunk(same, ke, ve, kw, vw, win_len=70), want)
    out = torch.full((2, 6, 8, 136), 7.0, device=cuda).half()
    assert ops.attn_chunk(q, ke, ve, kw, vw, win_len=70, out=out[..., :128].transpose(1, 2)).data_ptr() == out.data_ptr()
    assert torch.equal(out[..., :128].transpose(1, 2), want) and bool((out[..., 128:] == 7).all())
    odd.fill_(7)
    assert torch.equal(ops.attn_chunk(q, ke, ve, kw, vw, win_len=70, out=odd), want) and torch.equal(odd, want)
    shared = q[:, :1].expand(2, 8, 6, 128)
    assert torch.equal(ops.attn_chunk(shared, ke, ve, kw, vw, win_len=70), ops.attn_chunk(shared.contiguous(), ke, ve, kw, vw, win_len=70))


def test_a_longer_cache_row_and_streams_without_alignment(cuda):
    q, ke, ve, kw, vw = _case(cuda, 2, 8, 2, 6, 256, 70, torch.float16)
    want = ops.attn_chunk(q, ke, ve, kw, vw, win_len=70)
    for side in (ke, ve):
        side["tokens"] = 256
        for f in ("scale", "zero"):
            side[f] = torch.cat((side[f], torch.full((2, 128), float("nan"), device=cuda).half()), 1)
        moved = torch.empty(side["size"] + 2, dtype=torch.uint8, device=cuda)
        moved[2:] = side["stream"][:side["size"]]
        side["stream"] = moved[2:]
    assert torch.equal(ops.attn_chunk(q, ke, ve, kw, vw, win_len=70), want)


def test_a_few_tokens_agree_with_single_steps(cuda):
    """One query at a time through attn_decode over the same tokens is within both kernels' tolerance."""
    B, Hq, Hkv, n, T, W = 2, 32, 8, 4, 2048, 100
    q, ke, ve, kw, vw = _case(cuda, B, Hq, Hkv, n, T, W, torch.float16)
    got = ops.attn_chunk(q, ke, ve, kw, vw, win_len=W)
    for i in range(n):
        one = ops.attn_decode(q[:, :, i].contiguous(), ke, ve, kw, vw, win_len=W - n + 1 + i)
        assert (got[:, :, i].float() - one.float()).abs().max().item() < 1e-3


def test_damaged_block_info_is_survived(cuda):
    q, ke, ve, kw, vw = _case(cuda, 2, 8, 2, 6, 512, 70, torch.float16)
    g = torch.Generator(device=cuda).manual_seed(1)
    for side in (ke, ve):
        info = side["info"].view(torch.int32)
        info.copy_(torch.randint(-2 ** 31, 2 ** 31 - 1, info.shape, generator=g, device=cuda))
    ops.attn_chunk(q, ke, ve, kw, vw, win_len=70)
    for side in (ke, ve):                                  # in the buffer, but anywhere: headers and widths are noise
        info = side["info"].view(torch.int32)
        info.copy_(torch.randint(0, side["size"] // 2, info.shape, generator=g, device=cuda) * 2)
    ops.attn_chunk(q, ke, ve, kw, vw, win_len=70)
    torch.cuda.synchronize()


def test_two_streams_and_a_graph(cuda):
    B, Hq, Hkv, n, T, W = 2, 8, 2, 5, 2048, 60
    q, ke, ve, kw, vw = _case(cuda, B, Hq, Hkv, n, T, W, torch.bfloat16)
    want = ops.attn_chunk(q, ke, ve, kw, vw, win_len=W)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.attn_chunk(q, ke, ve, kw, vw, win_len=W))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = ops.attn_chunk(q, ke, ve, kw, vw, win_len=W)
        graphs.append((g, got))
    for step in range(3):
        q.copy_(torch.randn(q.shape, device=cuda))
        for g, _ in graphs:
            g.replay()
        want = ops.attn_chunk(q, ke, ve, kw, vw, win_len=W)
        torch.cuda.synchronize()
        assert all(torch.equal(got, want) for _, got in graphs)


def test_refusals(cuda):
    q, ke, ve, kw, vw = _case(cuda, 2, 8, 2, 6, 256, 70, torch.float16)

    def bad(match, **kw_):
        args = dict(q=q, k=ke, v=ve, k_win=kw, v_win=vw, win_len=70)
        args.update(kw_)
        with pytest.raises(RuntimeError, match=match):
            ops.attn_chunk(**args)

    bad("device tensor", q=q[:, :, 0])
    bad("device tensor", q=q.cpu())
    bad("Unsupported data type", q=q.float())
    bad("q's dtype", q=q.bfloat16())
    bad("go together", v=None)
    bad("go together", v_win=None)
    bad("empty cache", k=None, v=None, k_win=None, v_win=None)
    bad("empty cache", k=None, v=None, win_len=0)
    bad("win_len", win_len=321)
    bad("multiple of Hkv", q=q[:, :7])
    bad("multiple of 128", k=dict(ke, tokens=192), v=dict(ve, tokens=192))
    bad("different token counts", k=dict(ke, tokens=128))
    bad("block num", k=dict(ke, info=ke["info"][:4]))
    bad("head count", k_win=kw[:, :1].contiguous(), v_win=vw[:, :1].contiguous())
    bad("more queries", q=q.repeat(1, 1, 60, 1))
    bad("starts", starts=torch.zeros(2, device=cuda))
    bad("starts", starts=torch.zeros(2, dtype=torch.int32))
    bad("out must match", out=q.float())
    bad("share elements", out=q[:, :1].expand(2, 8, 6, 128))
    bad("on q's device", k=dict(ke, scale=ke["scale"].cpu()))
    bad("bits_len", k=dict(ke, bits=9))


def test_windows_and_queries_further_apart_than_32_bits(cuda):
    B, Hq, Hkv, n, W, cap = 2, 4, 2, 5, 150, (1 << 22) + 70
    q, _, _, kw, vw = _case(cuda, B, Hq, Hkv, n, 0, W, torch.float16, cap=W)
    want = ops.attn_chunk(q, None, None, kw, vw)
    big = [torch.empty(B, Hkv, cap, 128, dtype=torch.float16, device=cuda) for _ in range(2)]
    for far, near in zip(big, (kw, vw)):
        far[:, :, :W].copy_(near)
    flat = torch.empty((1 << 31) + 8192, dtype=torch.float16, device=cuda)
    far_q, out = (flat.as_strided(q.shape, (1 << 31, n * 128, 128, 1), at) for at in (0, 4096))
    far_q.copy_(q)
    assert torch.equal(ops.attn_chunk(far_q, None, None, *big, win_len=W, out=out), want) and torch.equal(out, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Hq,Hkv,n", [(8, 2, 4), (5, 1, 3), (8, 2, 5), (6, 6, 2), (17, 1, 1), (16, 1, 1)])
def test_few_rows_and_scales_of_far_apart_sizes(cuda, dtype, Hq, Hkv, n):
    """Up to and over sixteen rows a KV head, with and without the causal mask; values' scales that grow and fall over the tokens."""
    B, T, W = 2, 1024, 50
    q, ke, ve, kw, vw = _case(cuda, B, Hq, Hkv, n, T, W, dtype, seed=Hq + n)
    span = 2.0 ** torch.linspace(-9, 9, T, device=cuda)
    for order in (1, -1):
        ve2 = dict(ve, scale=(ve["scale"].float() * (span if order > 0 else span.flip(0))).to(dtype))
        q2 = q.clone()
        q2[:, 0] *= 7
        K, V, size = _values(ke, ve2, kw, vw, B, Hkv, W)
        co.check(ops.attn_chunk(q2, ke, ve2, kw, vw, win_len=W), q2, K, V, **size)
        co.check(ops.attn_chunk(q2, ke, ve2, kw, vw, win_len=W, causal=False, sm_scale=0.2), q2, K, V, causal=False, sm=0.2, **size)
