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


def _tile_bytes(B, Hkv, keys):
    return B * Hkv * -(-keys // 128) * 2 * 128 * 128 * 4  # sums of dV and dK of the key tiles


@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("B,Hq,Hkv,S,window,sinks", [
    (1, 24, 24, 30720, 128, 4096), (1, 24, 24, 30720, 1152, 4096), (1, 24, 24, 65536, 1024, 8192), (1, 24, 24, 65536, 128, 16384), (2, 32, 8, 32768, 512, 8192), (1, 24, 24, 30720, 128, 30720),
    (1, 24, 24, 69120, 128, 69120), (64, 16, 4, 4096, 64, 4096), (1, 24, 6, 1 << 20, 128, 1 << 16),
])
def test_workspace_of_many_sinks_is_bounded(causal, B, Hq, Hkv, S, window, sinks):
    """A tile with sinks leaves its own sums and those of one part of the rows outside of its window; beyond that there are as many parts as work-groups, four to a
    compute unit."""
    n = _load().fba_window_workspace_bytes(0, B, Hq, Hkv, S, S, window, sinks, causal)
    assert 0 < n <= 2 * _tile_bytes(B, Hkv, sinks) + _tile_bytes(1, 1, 4 * 256 * 128)


def test_workspace_of_few_sinks_is_what_it_was():
    lib = _load()
    assert lib.fba_window_workspace_bytes(0, 1, 24, 24, 30720, 30720, 1152, 384, 0) == 72 * 14 * 131072
    assert lib.fba_window_workspace_bytes(0, 1, 24, 6, 30720, 30720, 1536, 128, 1) == 6 * 19 * 131072
