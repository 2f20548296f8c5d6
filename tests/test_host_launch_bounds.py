"""Calls whose launch would have 2^32 threads or more, which HIP counts in 32 bits, are refused before it."""
import ctypes

from packkv_amd import _lib


def _status(call, a, *rest):
    return call(ctypes.byref(a), *rest, None), _lib.load().pkv_last_error()


def test_rotary():
    def status(n):
        a = _lib.RotaryArgs()
        for f in ("q", "k", "q_out", "k_out", "positions", "inv_freq"):
            setattr(a, f, 4096)
        a.dtype, a.B, a.Hq, a.Hkv, a.n, a.n_axes, a.pos_bytes = _lib.F16, 1, 8, 8, n, 1, 8
        return _status(_lib.load().pkv_norm_rotary, a)

    for n in ((1 << 26) - 3, 1 << 26, (1 << 31) - 1):      # a wavefront a token, four to a workgroup
        code, text = status(n)
        assert code == _lib.ERR_UNSUPPORTED and b"too large" in text, (n, code, text)


def test_sample():
    def status(rows):
        a = _lib.SampleArgs()
        a.logits = a.u = a.token = 4096
        a.dtype, a.rows, a.vocab, a.row_stride = _lib.F32, rows, 50, 0
        return _status(_lib.load().pkv_sample, a, None, 0)

    for rows in (1 << 22, (1 << 31) - 1):                  # a workgroup of 1024 a row
        code, text = status(rows)
        assert code == _lib.ERR_UNSUPPORTED and b"rows" in text, (rows, code, text)


def test_chunk():
    def status(n, Hq=1, bits=4):
        a = _lib.ChunkArgs()
        for f in ("k_stream", "k_info", "v_stream", "v_info", "k_scale", "k_zero", "v_scale", "v_zero", "q", "out"):
            setattr(a, f, 4096)
        a.k_bytes = a.v_bytes = 1 << 20
        a.B, a.Hq, a.Hkv, a.n, a.T_c, a.T_w, a.k_bits, a.v_bits, a.dtype, a.sm_scale = 1, Hq, 1, n, 1024, 0, bits, bits, _lib.BF16, 0.1
        return _status(_lib.load().pkv_attn_chunk, a, 4096, 1 << 50)

    for n, Hq, bits in (((1 << 27) - 100, 1, 4), (1 << 27, 1, 4), (1 << 26, 8, 4), (1 << 26, 1, 8)):     # 128 rows (at 8 bits 32), for 8 XCDs
        code, text = status(n, Hq, bits)
        assert code == _lib.ERR_UNSUPPORTED and b"too large" in text, (n, Hq, bits, code, text)
