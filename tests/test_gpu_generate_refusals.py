"""generate and forward: what they refuse, and that a refused call leaves the cache as it was."""
import pytest
import torch

from packkv_amd.decoder import DecoderShape, ShapedDecoder

pytestmark = pytest.mark.gpu

SHAPE = dict(layers=1, hidden=256, q_heads=4, kv_heads=2, mlp=512, vocab=640)


@pytest.fixture(scope="module")
def model(cuda):
    return ShapedDecoder(DecoderShape(**SHAPE), dtype=torch.float16, device=cuda, seed=3)


def _prompt(cuda, n=140, B=2):
    return torch.randint(1, 640, (B, n), generator=torch.Generator().manual_seed(n)).to(cuda)


def test_rows_without_a_token_are_no_result(cuda, model):
    """A sequence whose logits are NaN has no next token: generate says so instead of going on with another one's embedding."""
    ids, u = _prompt(cuda), torch.rand(4, 2, generator=torch.Generator().manual_seed(1)).to(cuda)
    model.generate(ids, model.new_cache(2, 512), u)
    kept = model.embed[0].clone()
    ids[1, -1] = 0
    try:
        model.embed[0] = float("nan")
        with pytest.raises(RuntimeError, match="nothing can be chosen"):
            model.generate(ids, model.new_cache(2, 512), u)
    finally:
        model.embed[0] = kept


def test_forward_refuses_unknown_ways(cuda, model, monkeypatch):
    cache, ids = model.new_cache(2, 512), _prompt(cuda)
    for way in ("one", "", None, "Fused"):
        with pytest.raises(RuntimeError, match="rotary"):
            model.forward(ids, cache, rotary=way)
    assert cache.get_seq_length() == 0


def test_one_pass_forms_no_tables(cuda, model, monkeypatch):
    """rotary="fused" turns rows by positions; the chain's cosines and sines are not formed beside it."""
    cache, ids = model.new_cache(2, 512), _prompt(cuda)
    calls = []
    tables = model._rotary
    monkeypatch.setattr(model, "_rotary", lambda *a: calls.append(a) or tables(*a))
    model.generate(ids, cache, torch.rand(3, 2, device=cuda))
    assert calls == [] and cache.get_seq_length() == 143
    model.forward(ids[:, :1], cache)
    assert len(calls) == 1


def test_generate_refuses_before_the_prompt_is_in_the_cache(cuda, model):
    cache, ids, u = model.new_cache(2, 512), _prompt(cuda), torch.rand(3, 2, device=cuda)
    for kw in (dict(u=u.double()), dict(u=u.cpu()), dict(u=u[:, :1]), dict(u=u[:, None]), dict(u=u[0]), dict(temperature=-1.0), dict(top_p=1.5),
               dict(top_k=-1), dict(min_p=torch.zeros(3, device=cuda)), dict(top_k=torch.zeros(2, device=cuda)), dict(temperature=torch.ones(2))):
        with pytest.raises(RuntimeError):
            model.generate(ids, cache, **{"u": u, **kw})
        assert cache.get_seq_length() == 0, kw
    want = model.generate(ids, cache, u, top_k=torch.full((2,), 9, dtype=torch.int32, device=cuda))
    assert torch.equal(model.generate(ids, model.new_cache(2, 512), (row for row in u), top_k=9), want)
