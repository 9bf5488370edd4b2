"""CPU: the argument checks of the quantised key/value cache (C ABI and Python) and the rotation's table; no GPU needed."""
import ctypes
import math

import pytest
import torch


def _args(**kw):
    from gemlite_b200 import _lib
    a = _lib.GLKvArgs()
    # never dereferenced: every call below is refused, or has nothing to do
    for n in ("k_codes", "v_codes", "k_scales", "v_scales", "page_table", "lens", "q", "k", "v", "out", "out_v"):
        setattr(a, n, 1 << 20)
    a.num_pages, a.page_size, a.n_kv_heads, a.n_q_heads, a.head_dim = 4, 16, 2, 4, 128
    a.batch, a.max_pages, a.n_tokens, a.max_len, a.max_new, a.x_dtype = 2, 2, 2, 32, 1, 2
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def test_struct_matches_the_header(lib):
    from gemlite_b200 import _lib
    # 20 pointers + 1 uint64 + 8 int64 (232) + 17 int32 + 2 floats + 1 int32 (80)
    assert ctypes.sizeof(_lib.GLKvArgs) == 312


@pytest.mark.parametrize("fn", ["gl_kv_write", "gl_kv_read", "gl_kv_attend"])
@pytest.mark.parametrize("bad", [{"format": 3}, {"format": -1}, {"num_pages": 0}, {"page_size": 0}, {"n_kv_heads": 0}, {"batch": -1},
                                 {"n_tokens": -1}, {"k_codes": None}, {"v_scales": None}, {"v_codes": (1 << 20) + 8}, {"lens": None},
                                 {"page_table": None}, {"n_tokens": 3}, {"format": 2}, {"max_len": -1}, {"out": (1 << 20) + 4}])
def test_bad_arguments_are_refused(lib, fn, bad):
    from gemlite_b200 import _lib
    assert getattr(lib, fn)(ctypes.byref(_args(**bad)), None) == _lib.GL_E_INVALID
    assert fn.encode() in lib.gl_last_error()


def test_unsupported_and_call_specific(lib):
    from gemlite_b200 import _lib
    for fn in ("gl_kv_write", "gl_kv_read", "gl_kv_attend"):
        f = getattr(lib, fn)
        assert f(ctypes.byref(_args(head_dim=96)), None) == _lib.GL_E_UNSUPPORTED
        assert f(ctypes.byref(_args(x_dtype=4)), None) == _lib.GL_E_UNSUPPORTED
        assert f(None, None) == _lib.GL_E_INVALID
        assert f(ctypes.byref(_args(batch=0, max_len=0, n_tokens=0)), None) == _lib.GL_OK
    for bad in ({"rot_dim": 24}, {"rot_dim": 144}, {"rot_dim": 64}, {"rot_dim": 64, "cos_sin": (1 << 20) + 4, "positions": 1 << 20, "table_rows": 4}, {"k": None}, {"q_stride_n": 4}, {"v": (1 << 20) + 2},
                {"q_norm": 1 << 20, "norm_dtype": 4}, {"n_q_heads": 0}):
        assert lib.gl_kv_write(ctypes.byref(_args(**bad)), None) == _lib.GL_E_INVALID, bad
    for bad in ({"n_q_heads": 3}, {"n_q_heads": 0}, {"q": None}, {"q_stride_h": 12}, {"mask": 1 << 20, "mask_cols": -1}, {"kernel_override": 3}):
        assert lib.gl_kv_attend(ctypes.byref(_args(**bad)), None) == _lib.GL_E_INVALID, bad
    assert lib.gl_kv_attend(ctypes.byref(_args(n_q_heads=1 << 16, n_kv_heads=1, n_tokens=1 << 16)), None) == _lib.GL_E_UNSUPPORTED
    assert lib.gl_kv_attend(ctypes.byref(_args(max_pages=1 << 28)), None) == _lib.GL_E_UNSUPPORTED
    for fn in ("gl_kv_write", "gl_kv_read", "gl_kv_attend"):       # slots are 32-bit numbers
        assert getattr(lib, fn)(ctypes.byref(_args(num_pages=1 << 26, page_size=64)), None) == _lib.GL_E_UNSUPPORTED
    long = _args(max_pages=1 << 12, max_len=1 << 16)
    need = lib.gl_kv_attend_workspace_bytes(ctypes.byref(long))
    assert need > 0 and need % 16 == 0
    assert lib.gl_kv_attend(ctypes.byref(long), None) == _lib.GL_E_WORKSPACE and str(need).encode() in lib.gl_last_error()


def test_python_refuses_cpu_tensors(lib):
    from gemlite_b200 import KVBatch, QuantizedKVCache
    with pytest.raises(RuntimeError):
        KVBatch(torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(RuntimeError):
        QuantizedKVCache(1, 16, 1, 64, "fp8", device="cpu")
    with pytest.raises(ValueError):
        QuantizedKVCache(1, 16, 1, 64, "int3", device="cpu")


def test_rotary_table():
    from gemlite_b200 import rotary_table
    t = rotary_table(70001, 64, 500000.0, device="cpu")
    assert t.shape == (70001, 64) and t.dtype == torch.float32
    for p in (0, 1, 4097, 70000):
        for i in (0, 5, 31):
            angle = p * 500000.0 ** (-2 * i / 64)
            assert abs(float(t[p, i]) - math.cos(angle)) < 1e-7 and abs(float(t[p, 32 + i]) - math.sin(angle)) < 1e-7
    for rot in (0, -2, 7):
        with pytest.raises(ValueError):
            rotary_table(4, rot, device="cpu")
