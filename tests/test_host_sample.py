"""Host side of sample: refusals before any launch, and the workspace."""
import ctypes

import pytest
import torch

from packkv_amd import _lib, ops


def _args(**kw):
    a = _lib.SampleArgs()
    a.logits = a.u = a.token = 4096
    a.dtype, a.rows, a.vocab, a.row_stride = _lib.F32, 2, 1000, 1000
    for f, x in kw.items():
        setattr(a, f, x)
    return a


def test_refusals_before_any_launch():
    lib = _lib.load()
    call = lambda ws=4096, size=1 << 40, **kw: lib.pkv_sample(ctypes.byref(_args(**kw)), ws, size, None)
    assert lib.pkv_sample(None, None, 0, None) == _lib.ERR_INVALID
    for f in ("logits", "u", "token"):
        assert call(**{f: None}) == _lib.ERR_INVALID
    for f, x in (("rows", 0), ("vocab", 0), ("row_stride", -1), ("logits", 4098)):
        assert call(**{f: x}) == _lib.ERR_INVALID, f
    for f, x in (("dtype", 3), ("vocab", (1 << 20) + 1)):
        assert call(**{f: x}) == _lib.ERR_UNSUPPORTED, f
    big = dict(vocab=151936, row_stride=151936)
    assert call(ws=None, **big) == _lib.ERR_CAPACITY and call(size=1000, **big) == _lib.ERR_CAPACITY and call(ws=4104, **big) == _lib.ERR_CAPACITY


def test_workspace_is_for_rows_that_are_cut():
    size = lambda **kw: _lib.load().pkv_sample_workspace(ctypes.byref(_args(**kw)))
    assert size() == 0 and size(rows=256, vocab=151936) == 0 and size(vocab=(1 << 20) + 1) == 0
    one = size(rows=1, vocab=151936)
    assert one % 16 == 0 and 0 < one < 1 << 18 and size(rows=3, vocab=151936) == 3 * one


def test_host_tensors_are_refused():
    with pytest.raises(RuntimeError, match="device tensor"):
        ops.sample(torch.zeros(1, 8), torch.zeros(1))
