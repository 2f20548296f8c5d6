"""The native host side of norm_rotary, window_append_rotary, attn_chunk and sample against the general code: the same bits where it
serves a call, and calls that it leaves alone get through."""
import pytest
import torch

from packkv_amd import _lib, ops, synth

pytestmark = pytest.mark.gpu


class _Counting:
    def __init__(self, host):
        self.host, self.served = host, []

    def __getattr__(self, name):
        def call(*args):
            got = getattr(self.host, name)(*args)
            self.served.append(got is not None)
            return got
        return call


def _both(monkeypatch, call, served=True):
    host = _Counting(_lib.host)
    monkeypatch.setattr(_lib, "host", host)
    got = call()
    assert host.served == [served], host.served
    monkeypatch.setattr(_lib, "host", _lib.NO_HOST)
    want = call()
    monkeypatch.setattr(_lib, "host", host.host)
    flat = lambda r: r if isinstance(r, tuple) else (r,)
    for a, b in zip(flat(got), flat(want)):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and torch.equal(a, b)
    return got


@pytest.fixture
def native(cuda):
    if _lib.host is _lib.NO_HOST:
        pytest.skip("the native host side is not built for this torch")
    return cuda


def test_rotary(native, monkeypatch):
    cuda = native
    x = torch.randn(3, 5, 24, 128, device=cuda).half()
    q, k, v = (t.transpose(1, 2) for t in x.split((16, 4, 4), dim=2))
    inv, w = torch.rand(64, device=cuda), torch.rand(128, device=cuda).half()
    pos = torch.randint(0, 1000, (3, 3, 5), device=cuda)
    for p, sec, inter in ((pos[0], None, False), (pos[0, 0], None, False), (pos[0, :, :1].int(), None, True), (pos, (16, 24, 24), False),
                          (pos[:, :1], (24, 20, 20), True), (pos[0, 0], (44, 20, 0), True), (pos[:1], (64,), False)):
        for qw, kw in ((w, w), (None, w), (None, None)):
            _both(monkeypatch, lambda: ops.norm_rotary(q, k, p, inv, qw, kw, 1e-5, sec, inter))
    windows = []

    def step():
        kw, vw = torch.zeros(3, 4, 40, 128, device=cuda).half(), torch.ones(3, 4, 40, 128, device=cuda).half()
        windows.append((kw, vw))
        return ops.window_append_rotary(q, k, v, pos, inv, kw, vw, 7, w, w, sections=(16, 24, 24))
    _both(monkeypatch, step)
    assert torch.equal(windows[0][0], windows[1][0]) and torch.equal(windows[0][1], windows[1][1])
    # left to the general code: channels apart, lists for tuples, whole numbers for eps
    _both(monkeypatch, lambda: ops.norm_rotary(q.transpose(2, 3).contiguous().transpose(2, 3), k, pos[0], inv), served=False)
    _both(monkeypatch, lambda: ops.norm_rotary(q, k, pos, inv, sections=[16, 24, 24]), served=False)
    _both(monkeypatch, lambda: ops.norm_rotary(q, k, pos[0], inv, w, w, 1), served=False)


def test_chunk(native, monkeypatch):
    cuda = native
    k, v = synth.make_kv(2, 2, 420, seed=3, device=cuda)
    ke, ve = ops.k_quant_encode(k[:, :, :384].contiguous(), 0.1), ops.v_quant_encode(v[:, :, :384].contiguous(), 0.1)
    kw, vw = k[:, :, 384:].contiguous(), v[:, :, 384:].contiguous()
    q = synth.make_q(2, 8, device=cuda)[:, None].repeat(1, 7, 1, 1).transpose(1, 2)
    st = torch.tensor([3, 400], dtype=torch.int32, device=cuda)
    for args in ((ke, ve, kw, vw), (ke, ve, None, None), (None, None, kw, vw)):
        _both(monkeypatch, lambda: ops.attn_chunk(q, *args))
        _both(monkeypatch, lambda: ops.attn_chunk(q.contiguous(), *args, sm_scale=0.2, starts=st, causal=False))
    _both(monkeypatch, lambda: ops.attn_chunk(q, ke, ve, kw, vw, win_len=9))
    _both(monkeypatch, lambda: ops.attn_chunk(q, ke, ve, kw, vw, sm_scale=1), served=False)
    _both(monkeypatch, lambda: ops.attn_chunk(q.transpose(2, 3).contiguous().transpose(2, 3), ke, ve), served=False)


def test_sample(native, monkeypatch):
    cuda = native
    x, u = torch.randn(6, 9001, device=cuda), torch.rand(6, device=cuda)
    row = lambda lo, hi: lo + (hi - lo) * torch.rand(6, device=cuda)
    for logits in (x, x.half(), x.bfloat16(), x[:, 1:], x[::2]):
        n = logits.size(0)
        for kw in (dict(), dict(temperature=0.5, top_k=7, top_p=0.8, min_p=0.01, want_logprob=True),
                   dict(temperature=row(0.1, 2.0)[:n], top_k=torch.arange(n, dtype=torch.int32, device=cuda), top_p=row(0.5, 1.0)[:n], min_p=row(0.0, 0.1)[:n])):
            _both(monkeypatch, lambda: ops.sample(logits, u[:n], **kw))
    _both(monkeypatch, lambda: ops.sample(x, u, top_p=1), served=False)
    _both(monkeypatch, lambda: ops.sample(x.t().contiguous().t(), u), served=False)
