"""sample's numbers are checked as they are given, before they are rounded to float32, whichever side serves the call."""
import pytest
import torch

from packkv_amd import _lib, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("with_out", [False, True])
def test_numbers_just_out_of_range(cuda, monkeypatch, native, with_out):
    if not native:
        monkeypatch.setattr(_lib, "host", _lib.NO_HOST)
    x, u = torch.randn(3, 500, device=cuda), torch.rand(3, device=cuda)
    out = torch.empty(3, dtype=torch.int64, device=cuda) if with_out else None
    for kw in (dict(top_p=1.00000001), dict(top_p=-1e-60), dict(min_p=1.00000001), dict(min_p=-1e-60), dict(temperature=-1e-60),
               dict(temperature=float("nan")), dict(top_p=float("nan")), dict(top_k=-1), dict(top_k=1 << 31)):
        with pytest.raises(RuntimeError, match="%s is out of range" % next(iter(kw))):
            ops.sample(x, u, out=out, **kw)
    want = ops.sample(x, u, temperature=0.0)
    for kw in (dict(temperature=1e-60), dict(temperature=-0.0), dict(top_p=1e-60), dict(top_k=1, temperature=1e300), dict(min_p=1.0)):
        assert torch.equal(ops.sample(x, u, out=out, **kw), want), kw
    assert torch.equal(ops.sample(x, u, top_p=0.999999999999), ops.sample(x, u))
