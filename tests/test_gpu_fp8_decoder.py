"""The decoder with projections in 8-bit floating point: every call that a prompt, a later prompt and single steps make, against 64 bits on the
call's own inputs, and the calls' order and wiring."""
import pytest
import torch

import fp8_oracle as oracle
from packkv_amd import ops
from packkv_amd.decoder import DecoderShape, ShapedDecoder
from test_gpu_fp8 import _check_norm

pytestmark = pytest.mark.gpu
SHAPE = dict(layers=2, hidden=400, q_heads=4, kv_heads=2, mlp=656, vocab=640)       # ragged blocks everywhere
ORDER = ["add_rms_norm", "fp8_linear", "fp8_quantize", "fp8_linear", "add_rms_norm", "fp8_gated", "fp8_quantize", "fp8_linear"]


def _rows(e):
    return {"codes": e["codes"].reshape(-1, e["codes"].size(-1)), "scale": e["scale"].reshape(-1, e["scale"].size(-1))}


@pytest.fixture
def calls(monkeypatch):
    """The 8-bit operators' calls as (name, arguments, keywords, result)."""
    made = []
    for name in set(ORDER):
        def call(*args, _name=name, _f=getattr(ops, name), **kw):
            made.append((_name, args, kw, _f(*args, **kw)))
            return made[-1][3]
        monkeypatch.setattr(ops, name, call)
    return made


def _check_call(name, args, kw, out, dtype):
    if name == "add_rms_norm":
        res = kw.get("residual")
        y, h = (out, None) if res is None else out
        _check_norm(args[0], args[1], args[2], res, y, h, dtype, kw["fp8"])
    elif name == "fp8_quantize":
        x = args[0].transpose(1, 2).flatten(2) if kw.get("heads") else args[0]
        assert out["codes"].shape == x.shape
        oracle.check_eight(out, x.reshape(-1, x.size(-1)).cpu().double(), 1)
    else:
        y, tol, var = oracle.product(_rows(args[0]), args[1])
        if name == "fp8_gated":
            n = y.size(1) // 2
            y, tol, var = oracle.gated(*((t[0], t[1], t[2]) for t in ((y[:, :n], tol[:, :n], var[:, :n]), (y[:, n:], tol[:, n:], var[:, n:]))))
        assert out.dtype == dtype
        oracle.check_rounded(out, y, tol, var)


@pytest.mark.parametrize("dtype,rotary", [(torch.float16, "chain"), (torch.bfloat16, "fused")])
def test_forward_call_by_call(cuda, calls, dtype, rotary):
    model = ShapedDecoder(DecoderShape(**SHAPE), dtype=dtype, device=cuda, seed=3, weights="fp8")
    s, B = model.shape, 2
    assert len(calls) == 4 * s.layers
    for name, args, kw, out in calls:
        assert name == "fp8_quantize" and kw == {"block": 128}
        oracle.check_eight(out, args[0].cpu().double(), 128)
    cache = model.new_cache(B, 1024)
    gen = torch.Generator().manual_seed(1)
    for n, attention in ((150, "dense"), (1, "fused"), (5, "fused"), (1, "dense")):
        del calls[:]
        ids = torch.randint(0, s.vocab, (B, n), generator=gen).to(cuda)
        taps = []
        logits = model.forward(ids, cache, attention=attention, rotary=rotary, taps=taps)
        assert logits.shape == (B, s.vocab) and logits.dtype == torch.float32 and bool(torch.isfinite(logits).all())
        assert [c[0] for c in calls] == ORDER * s.layers + ["add_rms_norm"]
        for c in calls:
            _check_call(*c, dtype)
        # what goes into each call is what came out of an earlier one
        h = model.embed[ids].view(B * n, s.hidden)
        more = None
        for li, blk in enumerate(model.blocks):
            norm1, qkv, quant, o, norm2, gated, quant2, down = calls[8 * li:8 * li + 8]
            if more is None:
                assert torch.equal(norm1[1][0], h) and norm1[2].get("residual") is None
                x = norm1[3]
            else:
                assert norm1[1][0] is more and torch.equal(norm1[2]["residual"], h)
                x, h = norm1[3]
            assert norm1[1][1] is blk["in_norm"] and qkv[1][0] is x and qkv[1][1] is blk["qkv"]
            assert torch.equal(quant[1][0], taps[li][1]) and quant[2] == {"heads": True}
            assert o[1][0] is quant[3] and o[1][1] is blk["o"]
            assert torch.equal(norm2[1][0], o[3].view(B * n, s.hidden)) and torch.equal(norm2[2]["residual"], h) and norm2[1][1] is blk["post_norm"]
            x, h = norm2[3]
            assert gated[1][0] is x and gated[1][1] is blk["gate_up"] and quant2[1][0] is gated[3] and down[1][0] is quant2[3] and down[1][1] is blk["down"]
            more = down[3]
        last = calls[-1]
        assert torch.equal(last[1][0], more.view(B, n, -1)[:, -1]) and torch.equal(last[2]["residual"], h.view(B, n, -1)[:, -1]) and last[1][1] is model.final_norm
        assert torch.equal(logits, torch.nn.functional.linear(last[3][0], model.lm_head).float())


def test_close_to_the_decoder_with_16_bit_weights(cuda):
    """Not a tolerance of the arithmetic (the calls' are above): a scale, an order or a residual gone wrong is off by one or more; e4m3's
    half step, 2^-4 of a value at most, 2.6 % in the mean, gives 4 % of a product, a few such in a row for the logits."""
    shape = DecoderShape(layers=2, hidden=512, q_heads=4, kv_heads=2, mlp=1024, vocab=640)
    eight, full = (ShapedDecoder(shape, device=cuda, seed=4, weights=w) for w in ("fp8", "same"))
    ids = torch.randint(0, 640, (2, 200), generator=torch.Generator().manual_seed(2)).to(cuda)
    a, b = (m.prefill(ids, m.new_cache(2, 512)) for m in (eight, full))
    assert float((a - b).norm() / b.norm()) < 0.25


def test_generate(cuda):
    model = ShapedDecoder(DecoderShape(**SHAPE), device=cuda, seed=3, weights="fp8")
    ids = torch.randint(0, 640, (3, 40), generator=torch.Generator().manual_seed(2)).to(cuda)
    u = torch.rand(12, 3, generator=torch.Generator().manual_seed(5)).to(cuda)
    got = [model.generate(ids, model.new_cache(3, 512), u, temperature=0.8, top_k=40) for _ in range(2)]
    assert got[0].shape == (3, 12) and torch.equal(got[0], got[1])
    assert model.greedy(ids, model.new_cache(3, 512), 4).shape == (3, 4)


def test_settings_are_refused():
    with pytest.raises(RuntimeError, match="not supported: weights"):
        ShapedDecoder(DecoderShape(**SHAPE), weights="int4", device="cpu")
