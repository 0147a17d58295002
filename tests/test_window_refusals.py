"""What window_attn_func and its C entry points refuse, without a GPU."""
import ctypes

import pytest
import torch


class Strided(ctypes.Structure):
    _fields_ = [("ptr", ctypes.c_void_p), ("batch", ctypes.c_int64), ("head", ctypes.c_int64), ("row", ctypes.c_int64)]


def _lib():
    from flex_block_attn_amd import _lib

    return _lib


GOOD = dict(B=1, Hq=2, Hkv=1, Sq=64, Skv=64, D=128, window=8, sinks=1, causal=1, type=0)


def _fwd(q=(0x1000, 128 * 64 * 2, 128 * 64, 128), lengths=None, stats=0x1000, **change):
    a = dict(GOOD, **change)
    t = [ctypes.byref(Strided(*x)) if x is not None else None for x in (q, *[(0x1000, 8192, 8192, 128)] * 3)]
    return _lib().load().fba_window_fwd(*t, None, ctypes.c_void_p(stats), ctypes.c_void_p(lengths), a["B"], a["Hq"], a["Hkv"], a["Sq"], a["Skv"], a["D"], a["window"], a["sinks"],
                                        a["causal"], a["type"], None)


@pytest.mark.parametrize("change,code,text", [
    (dict(D=64), 1, "head_dim"), (dict(type=2), 1, "type"), (dict(B=0), 1, "positive"), (dict(Skv=0), 1, "positive"), (dict(Hq=3, Hkv=2), 1, "multiple of Hkv"),
    (dict(window=0), 1, "window"), (dict(window=-1), 1, "window"), (dict(sinks=-1), 1, "sinks"), (dict(lengths=0x1000, Sq=32), 1, "lengths"),
    (dict(Sq=1 << 29), 2, "2^28"), (dict(Hq=1 << 12, Sq=1 << 20), 2, "2^29"), (dict(stats=None), 1, "stats"),
    (dict(q=None), 1, "q is null"), (dict(q=(0x1008, 0, 0, 128)), 1, "aligned"), (dict(q=(0x1000, 0, 0, 132)), 1, "strides"), (dict(q=(0x1000, 0, 0, -128)), 1, "strides"),
    (dict(q=(0x1000, 0, 0, 1 << 25)), 2, "rows may be"),
])
def test_c_entry_refuses(change, code, text):
    lib = _lib()
    assert _fwd(**change) == code
    assert text in lib.load().fba_last_error().decode()


def test_workspace_is_asked_for_and_checked():
    lib = _lib().load()
    assert lib.fba_window_workspace_bytes(0, 1, 1, 1, 64, 64, 64, 8, 1) == 0  # the window reaches over everything
    assert lib.fba_window_workspace_bytes(0, 1, 1, 1, 64, 64, 8, 0, 1) == 0   # no sinks
    n = lib.fba_window_workspace_bytes(0, 2, 3, 3, 1000, 1000, 8, 130, 1)
    assert n > 0 and n % (2 * 3 * 2 * 32 * 128 * 4) == 0  # batch, kv heads, dV and dK, 32 keys
    assert lib.fba_window_workspace_bytes(0, 1, 1, 1, 64, 64, 0, 0, 1) == -1
    t = ctypes.byref(Strided(0x1000, 1000 * 128, 1000 * 128, 128))
    f = ctypes.c_void_p(0x1000)
    args = (1, 1, 1, 1000, 1000, 128, 8, 4, 1, 0, None)
    assert lib.fba_window_bwd(t, t, t, t, None, t, f, None, t, t, t, None, 0, *args) == 1
    assert "ws must" in lib.fba_last_error().decode()
    assert lib.fba_window_bwd(t, t, t, t, None, t, f, None, t, t, t, f, 1000, *args) == 1
    other = ctypes.byref(Strided(0x1000, 1000 * 256, 1000 * 256, 256))
    assert lib.fba_window_bwd(t, t, t, t, None, other, f, None, t, t, t, f, 1 << 40, *args) == 2
    assert "row stride" in lib.fba_last_error().decode()


def test_python_refuses():
    import flex_block_attn_amd as fba

    q = torch.zeros((1, 2, 8, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU tensor"):
        fba.window_attn_func(q, q, q, 4)
    with pytest.raises(ValueError, match="GPU tensor"):
        fba.window_attn_func(q.float(), q, q, 4)


@pytest.mark.gpu
def test_python_refuses_on_the_gpu(gpu):
    import flex_block_attn_amd as fba

    new = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype, device=gpu)
    q, k = new(1, 4, 8, 128), new(1, 2, 8, 128)
    n = torch.tensor([8], dtype=torch.int32, device=gpu)
    for error, text, args, more in [
        (TypeError, "bfloat16 or float16", (q.float(), k, k, 4), {}),
        (ValueError, "type and device", (q, k.half(), k, 4), {}),
        (ValueError, "GPU tensor", (q, k, k.cpu(), 4), {}),
        (ValueError, "shape", (q[0], k, k, 4), {}),
        (ValueError, "head_dim", (new(1, 4, 8, 64), new(1, 2, 8, 64), new(1, 2, 8, 64), 4), {}),
        (ValueError, "batch", (q, new(2, 2, 8, 128), new(2, 2, 8, 128), 4), {}),
        (ValueError, "same shape", (q, k, new(1, 2, 9, 128), 4), {}),
        (ValueError, "multiple of kv heads", (q, new(1, 3, 8, 128), new(1, 3, 8, 128), 4), {}),
        (ValueError, "window", (q, k, k, 0), {}),
        (TypeError, "window", (q, k, k, 1.5), {}),
        (TypeError, "window", (q, k, k, True), {}),
        (ValueError, "sinks", (q, k, k, 4), dict(sinks=-1)),
        (TypeError, "sinks", (q, k, k, 4), dict(sinks=None)),
        (ValueError, "lengths", (q, k, k, 4), dict(lengths=n.long())),
        (ValueError, "lengths", (q, k, k, 4), dict(lengths=n[:0])),
        (ValueError, "lengths", (q, new(1, 2, 9, 128), new(1, 2, 9, 128), 4), dict(lengths=n)),
        (ValueError, "GPU tensor", (q, k, k, 4), dict(lengths=n.cpu())),
    ]:
        with pytest.raises(error, match=text):
            fba.window_attn_func(*args, **more)
    # wider numbers than 32 bits are windows over everything
    assert torch.equal(fba.window_attn_func(q, k, k, 1 << 40, sinks=1 << 40), fba.window_attn_func(q, k, k, None))
