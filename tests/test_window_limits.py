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


def _forward(B, Hq, Sq, Hkv=1, Skv=16):
    t = ctypes.byref(Strided(0x1000, 128, 128, 128))
    return _load().fba_window_fwd(t, t, t, t, None, A, None, B, Hq, Hkv, Sq, Skv, 128, 8, 1, 1, 0, None)


def _backward(B, Hq, Hkv, Sq, Skv, window=8, sinks=1):
    t = ctypes.byref(Strided(0x1000, 128, 128, 128))
    return _load().fba_window_bwd(t, t, t, t, None, t, A, None, t, t, t, A, 1 << 62, B, Hq, Hkv, Sq, Skv, 128, window, sinks, 1, 0, None)


def test_more_work_groups_than_a_launch_has_are_refused():
    """With the stated error, and before anything is launched."""
    lib = _load()
    for call in (lambda: _forward(1 << 24, 1, 1), lambda: _forward(1 << 20, 16, 3), lambda: _forward(1 << 22, 8, 15, 8, 15), lambda: _backward(1 << 24, 1, 1, 1, 1, sinks=0),
                 lambda: _backward(1 << 21, 8, 8, 1, 16), lambda: _backward(1 << 19, 1, 1, 16, 16)):
        assert call() == 2
        assert "launch" in lib.fba_last_error().decode()
    # sums of several parts, 32 work-groups to a tile: the workspace says so already
    assert lib.fba_window_workspace_bytes(0, 1 << 19, 1, 1, 16, 16, 8, 1, 1) == -1 and "launch" in lib.fba_last_error().decode()
    assert lib.fba_window_workspace_bytes(0, (1 << 19) - 1, 1, 1, 16, 16, 8, 1, 1) == ((1 << 19) - 1) * 2 * 131072
    assert lib.fba_window_workspace_bytes(0, 1 << 19, 1, 1, 16, 16, 16, 1, 1) == 0  # a window over everything: one part each


def test_more_work_groups_than_a_launch_has_are_refused_by_the_cache():
    lib = _load()

    class Cache(ctypes.Structure):
        _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "positions", "weights", "table", "lengths")] + [("pages", ctypes.c_int64)] + [
            (n, ctypes.c_int32) for n in ("kv_heads", "page_size", "batch", "max_pages")]

    t, much = ctypes.byref(Strided(0x1000, 128, 128, 128)), 1 << 62
    of = lambda batch, kv_heads, max_pages: ctypes.byref(Cache(*[0x1000] * 6, 10, kv_heads, 16, batch, max_pages))
    for call in (lambda: lib.fba_cache_attn(of(1 << 20, 1, 4), t, t, 16, 1 << 30, 0, 0, 0, A, much, None), lambda: lib.fba_cache_attn(of(1 << 10, 16, 1 << 16), t, t, 16, 1 << 30, 0, 1, 0, A, much, None),
                 lambda: lib.fba_cache_append(of((1 << 24) - 8000, 1, 4), t, t, None, None, None, 1, ctypes.c_void_p(0x2000), None)):
        assert call() == 2
        assert "too many" in lib.fba_last_error().decode() or "launch" in lib.fba_last_error().decode()
    assert lib.fba_cache_attn_workspace_bytes(of(1 << 20, 1, 4), 15, 0) > 0 and lib.fba_cache_attn_workspace_bytes(of(1 << 10, 16, 1 << 15), 16, 1) > 0
