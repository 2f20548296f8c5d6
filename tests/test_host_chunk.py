"""Host side of attn_chunk: what the entry point refuses before any launch, and its workspace."""
import ctypes

from packkv_amd import _lib


def _args(**kw):
    a = _lib.ChunkArgs()
    for f in ("k_stream", "k_info", "v_stream", "v_info", "k_scale", "k_zero", "v_scale", "v_zero", "q", "out", "k_win", "v_win"):
        setattr(a, f, 4096)
    a.k_bytes = a.v_bytes = 1 << 20
    a.B, a.Hq, a.Hkv, a.n, a.T_c, a.T_w, a.k_bits, a.v_bits, a.dtype, a.causal, a.sm_scale = 1, 32, 8, 4, 1024, 64, 4, 4, _lib.F16, 1, 0.1
    for f, x in kw.items():
        setattr(a, f, x)
    return a


def test_refusals_before_any_launch():
    lib = _lib.load()
    call = lambda ws=4096, size=1 << 40, **kw: lib.pkv_attn_chunk(ctypes.byref(_args(**kw)), ws, size, None)
    assert lib.pkv_attn_chunk(None, None, 0, None) == _lib.ERR_INVALID
    for f in ("q", "out", "k_stream", "v_info", "k_scale", "v_zero", "k_win", "v_win"):
        assert call(**{f: None}) == _lib.ERR_INVALID, f
    for f in ("q", "out", "k_stream", "v_stream", "k_win", "v_win"):
        assert call(**{f: 4098}) == _lib.ERR_INVALID and b"16-byte" in lib.pkv_last_error(), f
    for f, x in (("B", 0), ("Hkv", 0), ("n", 0), ("Hq", 0), ("Hq", 33), ("T_c", 100), ("T_c", -128), ("T_w", -1), ("n", 1089), ("par_stride", 1000),
                 ("win_stride", 60), ("k_bytes", 0), ("v_bytes", (1 << 32) - 4)):
        assert call(**{f: x}) == _lib.ERR_INVALID, (f, x)
    assert call(T_c=0, T_w=0) == _lib.ERR_INVALID
    for f, x in (("dtype", 2), ("k_bits", 1), ("v_bits", 9), ("B", 1 << 24)):
        assert call(**{f: x}) == _lib.ERR_UNSUPPORTED, (f, x)
    assert call(ws=None) == _lib.ERR_CAPACITY and call(size=100) == _lib.ERR_CAPACITY and call(ws=4104) == _lib.ERR_CAPACITY
    a = _args()
    a.q_stride[1] = 4
    assert lib.pkv_attn_chunk(ctypes.byref(a), 4096, 1 << 40, None) == _lib.ERR_INVALID


def test_workspace_holds_a_partial_for_each_row_and_run():
    lib = _lib.load()
    size = lambda **kw: lib.pkv_attn_chunk_workspace(ctypes.byref(_args(**kw)))
    assert size() % (32 * 4 * 132 * 4) == 0 and size() // (32 * 4 * 132 * 4) == 9      # 9 tiles, a run each
    assert size(n=1024, B=16) == 0                         # enough workgroups without
    assert size(T_c=128, T_w=0, n=1) == 0                  # one tile
    assert size(T_c=100) == 0                              # refused
