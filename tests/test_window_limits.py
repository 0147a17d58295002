"""What the C entries of window attention say about sizes and workspaces, without a GPU."""
import ctypes

import pytest


class Strided(ctypes.Structure):
    _fields_ = [("ptr", ctypes.c_void_p), ("batch", ctypes.c_int64), ("head", ctypes.c_int64), ("row", ctypes.c_int64)]


def _load():
    from flex_block_attn_amd import _lib

    return _lib.load()


A = ctypes.c_void_p(0x1000)


@pytest.mark.parametrize("lse,scratch", [(None, A), (A, None)])
def test_backward_with_statistics_of_its_own_refuses_null(lse, scratch):
    lib = _load()
    t = ctypes.byref(Strided(0x1000, 1000 * 128, 1000 * 128, 128))
    assert lib.fba_window_bwd_apart(t, t, t, t, None, t, lse, scratch, None, t, t, t, A, 1 << 40, 1, 1, 1, 1000, 1000, 128, 8, 4, 1, 0, None) == 1
    assert "lse or scratch" in lib.fba_last_error().decode()
