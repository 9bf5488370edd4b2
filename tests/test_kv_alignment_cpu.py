"""CPU: pointers that are not aligned to their element are refused at the C entries, before anything is launched."""
import ctypes

import pytest

from tests.test_kv_cache_cpu import _args


@pytest.mark.parametrize("fn", ["gl_kv_write", "gl_kv_read", "gl_kv_attend"])
@pytest.mark.parametrize("name", ["k_scales", "v_scales", "page_table", "lens", "q_offsets"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_four_byte_operands(lib, fn, name, off):
    from gemlite_b200 import _lib
    # (n_tokens = 0, max_len = 0: there is nothing to do once the arguments have passed)
    assert getattr(lib, fn)(ctypes.byref(_args(n_tokens=0, max_len=0)), None) == _lib.GL_OK
    assert getattr(lib, fn)(ctypes.byref(_args(n_tokens=0, max_len=0, **{name: (1 << 20) + off})), None) == _lib.GL_E_INVALID
    assert b"aligned" in lib.gl_last_error()


@pytest.mark.parametrize("bad", [{"q_norm": (1 << 20) + 2, "norm_dtype": 0}, {"k_norm": (1 << 20) + 1, "norm_dtype": 2}, {"k_norm": (1 << 20) + 1, "norm_dtype": 1},
                                 {"rot_dim": 64, "cos_sin": 1 << 20, "table_rows": 4, "positions": (1 << 20) + 2}])
def test_write_operands(lib, bad):
    from gemlite_b200 import _lib
    assert lib.gl_kv_write(ctypes.byref(_args(**bad)), None) == _lib.GL_E_INVALID
    assert b"misaligned" in lib.gl_last_error()


def test_status_needs_a_place_for_its_answer(lib):
    from gemlite_b200 import _lib
    assert lib.gl_kv_attend_status(None, 0, None) == _lib.GL_E_INVALID
    assert b"gl_kv_attend_status" in lib.gl_last_error()
