"""Host side of norm_rotary / window_append_rotary: refusals and the layout of the frequencies, without a GPU."""
import ctypes

import pytest
import torch

from packkv_amd import _lib, ops


def test_frequency_axes():
    assert ops._frequency_axes(None, False) == bytes(64)
    assert ops._frequency_axes((16, 24, 24), False) == bytes([0] * 16 + [1] * 24 + [2] * 24)
    got = ops._frequency_axes((24, 20, 20), True)
    assert [got.count(a) for a in (0, 1, 2)] == [24, 20, 20]
    assert all(got[i] == i % 3 for i in range(60)) and got[60:] == bytes(4)
    assert ops._frequency_axes((32, 32), True) == bytes([0, 1] * 32)
    assert ops._frequency_axes((64, 0, 0), True) == bytes(64)
    for bad, inter in (((16, 24, 23), False), ((16, 24, 24), True), ((), False), ((8,) * 8, False), ((80, -16), False)):
        with pytest.raises(RuntimeError, match="Assertion failed"):
            ops._frequency_axes(bad, inter)


def test_host_tensors_are_refused():
    q, k = torch.zeros(1, 4, 2, 128, dtype=torch.float16), torch.zeros(1, 2, 2, 128, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.norm_rotary(q, k, torch.zeros(1, 2, dtype=torch.int64), torch.ones(64))


def test_entry_point_checks_its_arguments():
    lib = _lib.load()

    def status(**kw):
        a = _lib.RotaryArgs()
        for f in ("q", "k", "q_out", "k_out", "positions", "inv_freq"):
            setattr(a, f, 4096)
        a.dtype, a.B, a.Hq, a.Hkv, a.n, a.n_axes, a.pos_bytes = _lib.F16, 1, 4, 2, 3, 1, 8
        for f, x in kw.items():
            if f == "axis0":
                a.axis[0] = x
            else:
                setattr(a, f, x)
        return lib.pkv_norm_rotary(ctypes.byref(a), None), lib.pkv_last_error()

    assert lib.pkv_norm_rotary(None, None) == _lib.ERR_INVALID
    for f in ("q", "k", "q_out", "k_out", "positions", "inv_freq"):
        assert status(**{f: None})[0] == _lib.ERR_INVALID
    assert status(v=4096) == (_lib.ERR_INVALID, b"values need an output, and an output values")
    assert status(v_out=4096)[0] == _lib.ERR_INVALID
    assert status(dtype=2)[0] == _lib.ERR_UNSUPPORTED
    for f in ("B", "Hq", "Hkv", "n"):
        assert status(**{f: 0})[0] == _lib.ERR_INVALID and status(**{f: -1})[0] == _lib.ERR_INVALID
    assert status(pos_bytes=2)[0] == _lib.ERR_INVALID
    assert status(n_axes=5)[0] == _lib.ERR_UNSUPPORTED and status(n_axes=0)[0] == _lib.ERR_UNSUPPORTED
    assert status(axis0=1)[0] == _lib.ERR_INVALID and b"axis" in status(axis0=1)[1]
    assert status(B=1 << 30, n=1 << 30)[0] == _lib.ERR_UNSUPPORTED
