"""The operators together, as a program that generates uses them: raw projections into the cache (update_rotary), attention of one
and of several new tokens (attend), sampled tokens (generate)."""
import pytest
import torch

import chunk_oracle as co
from packkv_amd import ops, synth
from packkv_amd.cache import PackKVCache, PackKVCacheConfig, PackKVCompressedCache
from packkv_amd.decoder import DecoderShape, ShapedDecoder

pytestmark = pytest.mark.gpu


def _values(cache, layer):
    L = cache.layers[layer]
    k, v = (side.as_dict() if side.tokens else None for side in (L.k, L.v))
    B, H = L.k_win.shape[:2]
    K, sizes = co.values_of(k, True, B, H, L.k_win, L.win_len)
    V, v_sizes = co.values_of(v, False, B, H, L.v_win, L.win_len)
    return K, V, dict(sizes=sizes, v_sizes=v_sizes)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("axes", [None, (16, 24, 24)])
def test_cache_through_prompts_and_steps(cuda, dtype, axes):
    """A prompt, single steps, drafts of several tokens and a second prompt, across cuts: the cache equals one that is given rotated
    keys, and every attend follows attention in 64 bits on what the cache holds."""
    B, Hq, Hkv = 2, 8, 2
    cfg = dict(max_tokens=2048, dtype=dtype, device=cuda)
    got, want = (PackKVCompressedCache(B, Hkv, 128, 1, PackKVCacheConfig(), **cfg) for _ in range(2))
    g = torch.Generator(device=cuda).manual_seed(2)
    inv = 1.0 / (1.0e6 ** (torch.arange(0, 128, 2, device=cuda, dtype=torch.float32) / 128))
    w = (1 + 0.2 * torch.randn(128, generator=g, device=cuda)).to(dtype)
    pos = 0
    for n in (300, 1, 1, 5, 17, 1, 64, 40, 1, 200, 1, 130, 3):
        qkv = torch.randn(B, n, Hq + 2 * Hkv, 128, generator=g, device=cuda).to(dtype)
        q, k, v = (x.transpose(1, 2) for x in qkv.split((Hq, Hkv, Hkv), dim=2))
        at = torch.arange(pos, pos + n, device=cuda)
        if axes:
            at = torch.stack((at, at + 7, 2 * at))[:, None]
        rq = got.update_rotary(q, k, v, 0, at, inv, w, w, 1e-5, axes)
        wq, wk = ops.norm_rotary(q, k, at, inv, w, w, 1e-5, axes)
        want.update(wk, v, 0, return_dense=False)
        pos += n
        assert torch.equal(rq, wq) and got.get_seq_length() == want.get_seq_length() == pos
        assert all(torch.equal(a, b) for a, b in zip(got.materialize(0), want.materialize(0)))
        K, V, sizes = _values(got, 0)
        out = got.attend(rq, 0)
        assert out.shape == rq.shape
        co.check(out, rq, K, V, **sizes)
        starts = torch.tensor([pos // 3, pos - n // 2], dtype=torch.int32, device=cuda)
        co.check(got.attend(rq, 0, starts=starts), rq, K, V, starts=starts.tolist(), **sizes)
    assert got.layers[0].k.tokens == 512


def test_attend_of_several_tokens_refuses_and_passes_on(cuda):
    k, v = synth.make_kv(1, 2, 300, seed=1, device=cuda)
    c = PackKVCache(1, 2, 128, 1, PackKVCacheConfig(), 1024)
    c.update(k, v, 0, return_dense=False)
    q = synth.make_q(1, 8, device=cuda).unsqueeze(2).repeat(1, 1, 5, 1)
    got = c.attend(q, 0, sm_scale=0.1)
    out = torch.empty_like(q)
    assert c.attend(q, 0, sm_scale=0.1, out=out) is out and torch.equal(out, got)
    one = torch.zeros(1, dtype=torch.int32, device=cuda)
    assert c.attend(q[:, :, 0], 0, starts=one).shape == (1, 8, 128)
    for kw in (dict(variant=1), dict(out_f32=True), dict(ref_rounding=True, variant=1)):
        with pytest.raises(RuntimeError, match="not supported"):
            c.attend(q, 0, **kw)
    with pytest.raises(RuntimeError, match="more queries"):
        c.attend(q.repeat(1, 1, 100, 1), 0)


@pytest.mark.parametrize("dtype,head_norm", [(torch.float16, False), (torch.bfloat16, True)])
def test_decoder_with_one_pass_rotary_and_later_prompts(cuda, dtype, head_norm):
    """Logits of the decoder with fused rotary and attention against the chain of library operators and dense attention, over a
    prompt, steps and a second prompt; the fused attention of the second prompt's layer 0 against 64 bits.  (The two decoders'
    layers quantise slightly different keys: logits are compared in norm, as for single steps.)"""
    shape = DecoderShape(layers=3, hidden=256, q_heads=4, kv_heads=2, mlp=512, vocab=640, head_norm=head_norm)
    model = ShapedDecoder(shape, dtype=dtype, device=cuda, seed=5)
    g = torch.Generator().manual_seed(6)
    a, b = model.new_cache(2, 1024), model.new_cache(2, 1024)
    for n in (330, 1, 1, 77, 1, 9, 1, 200):
        ids = torch.randint(0, shape.vocab, (2, n), generator=g).to(cuda)
        taps, later = [], a.get_seq_length() > 0
        la = model.forward(ids, a, attention="fused", taps=taps, rotary="fused")
        lb = model.forward(ids, b, attention="dense")
        assert ((la - lb).norm() / lb.norm()).item() < 0.05, n
        if later:
            K, V, sizes = _values(a, 0)
            co.check(taps[0][1], taps[0][0], K, V, sm=128 ** -0.5, **sizes)


def test_generate_samples_what_forward_says(cuda):
    """Tokens are those ops.sample gives for the logits of the same forwards; the cache holds them; a second prompt goes on."""
    shape = DecoderShape(layers=2, hidden=256, q_heads=8, kv_heads=2, mlp=512, vocab=4099, rope_sections=(24, 20, 20), rope_interleaved=True)
    model = ShapedDecoder(shape, dtype=torch.bfloat16, device=cuda, seed=7)
    g = torch.Generator().manual_seed(8)
    a, b = model.new_cache(3, 1024), model.new_cache(3, 1024)
    kw = dict(temperature=0.9, top_k=200, top_p=0.95, min_p=0.001)
    for n, steps in ((256, 20), (33, 70)):
        ids, u = torch.randint(0, shape.vocab, (3, n), generator=g).to(cuda), torch.rand(steps, 3, generator=g).to(cuda)
        got = model.generate(ids, a, u, **kw)
        logits = model.forward(ids, b, attention="fused" if b.get_seq_length() else "dense", rotary="fused")
        for i in range(steps):
            assert torch.equal(ops.sample(logits, u[i], **kw), got[:, i]), i
            logits = model.forward(got[:, i:i + 1], b, rotary="fused")
        assert a.get_seq_length() == b.get_seq_length()
    assert torch.equal(model.generate(ids, model.new_cache(3, 512), u[:3], temperature=0.0),
                       model.generate(ids, model.new_cache(3, 512), 0 * u[:3], top_k=1))
    assert model.generate(ids, model.new_cache(3, 512), u[:0]).shape == (3, 0)
    with pytest.raises(RuntimeError, match="rotary"):
        model.forward(ids, a)


def test_a_step_in_a_graph(cuda):
    """update_rotary's launch, attention of several tokens and sampling captured together and replayed."""
    B, Hq, Hkv, n, dtype = 2, 8, 2, 3, torch.float16
    k, v = synth.make_kv(B, Hkv, 520, seed=3, dtype=dtype, device=cuda)
    c = PackKVCompressedCache(B, Hkv, 128, 1, max_tokens=1024, dtype=dtype, device=cuda)
    c.update(k, v, 0, return_dense=False)
    L = c.layers[0]
    g = torch.Generator(device=cuda).manual_seed(4)
    x = torch.randn(B, n, Hq + 2 * Hkv, 128, generator=g, device=cuda).to(dtype)
    q, kn, vn = (t.transpose(1, 2) for t in x.split((Hq, Hkv, Hkv), dim=2))
    pos, inv = torch.arange(520, 520 + n, device=cuda), 1.0 / (1.0e6 ** (torch.arange(0, 128, 2, device=cuda, dtype=torch.float32) / 128))
    proj = torch.randn(Hq * 128, 9001, generator=g, device=cuda).to(dtype)
    u, row = torch.rand(B * n, generator=g, device=cuda), L.win_len

    def step():
        rq = ops.window_append_rotary(q, kn, vn, pos, inv, L.k_win, L.v_win, row)
        a = ops.attn_chunk(rq, L.k.as_dict(), L.v.as_dict(), L.k_win, L.v_win, win_len=row + n)
        return a, ops.sample(a.transpose(1, 2).reshape(B * n, -1) @ proj, u, top_k=30, top_p=0.9)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, tok = step()
    for _ in range(3):
        x.copy_(torch.randn(x.shape, generator=g, device=cuda))
        u.uniform_()
        graph.replay()
        torch.cuda.synchronize()
        got = a.clone(), tok.clone()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
