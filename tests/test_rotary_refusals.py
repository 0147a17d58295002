"""What rotary positions, the cache's rotation, its 4 bits and its rows read back refuse, and what `rotary` and `grid_coordinates` make, without a GPU."""
import ctypes
import math
from fractions import Fraction

import pytest
import torch

from test_cache_refusals import GOOD, Cache, Strided

A = 0x1000
ROW = Strided(A, 256, 128, 128)


class Cache4(ctypes.Structure):
    _fields_ = [("cache", Cache), ("k_scales", ctypes.c_void_p), ("v_scales", ctypes.c_void_p)]


class Rotation(ctypes.Structure):
    _fields_ = [("turns", ctypes.c_void_p), ("axes", ctypes.c_void_p), ("at", ctypes.c_void_p), ("at_batch", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in ("pairs", "n_axes", "interleaved")]


def _rotation(**change):
    return ctypes.byref(Rotation(**dict(dict(turns=A, axes=A, at=A, at_batch=0, pairs=64, n_axes=3, interleaved=1), **change)))


def _cache4(scales=A, **change):
    return ctypes.byref(Cache4(Cache(**dict(GOOD, **change)), scales, A))


def _lib():
    from flex_block_attn_amd import _lib

    return _lib.load()


BAD_ROTATIONS = [(dict(turns=None), "turns or axes"), (dict(axes=None), "turns or axes"), (dict(turns=A + 4), "aligned"), (dict(axes=A + 2), "aligned"), (dict(at=A + 1), "aligned"),
                 (dict(pairs=0), "pairs"), (dict(pairs=12), "pairs"), (dict(pairs=72), "pairs"), (dict(n_axes=0), "n_axes"), (dict(n_axes=9), "n_axes"), (dict(at_batch=-1), "at_batch")]


@pytest.mark.parametrize("change,text", BAD_ROTATIONS)
def test_c_entries_refuse_a_rotation(change, text):
    lib, q, out, r = _lib(), ctypes.byref(ROW), ctypes.c_void_p(0x2000), _rotation(**change)
    cache = ctypes.byref(Cache(**GOOD))
    for call in (lambda: lib.fba_rotary(q, q, None, None, r, 0, 1, 1, 0, 1, 128, 0, None), lambda: lib.fba_cache_append_rotary(cache, q, q, None, None, 0, r, None, None, None, 1, 0, out, None),
                 lambda: lib.fba_cache4_append(_cache4(), q, q, None, None, 0, r, None, None, None, 1, 0, out, None)):
        assert call() == 1 and text in lib.fba_last_error().decode()


def test_c_entries_refuse_arguments():
    lib, q, out, f, r, c, c4, odd = (_lib(), ctypes.byref(ROW), ctypes.c_void_p(0x2000), ctypes.c_void_p(A), _rotation(), ctypes.byref(Cache(**GOOD)), _cache4(), ctypes.byref(Strided(A, 4, 0, 128)))
    turn = lambda q=q, o=q, k=None, ko=None, r=r, B=1, Hq=1, Hk=0, S=1, D=128, t=0: lib.fba_rotary(q, o, k, ko, r, 0, B, Hq, Hk, S, D, t, None)
    append = lambda c=c, k=q, v=q, x=None, xo=None, heads=0, r=r, tokens=1, t=0, out=out: lib.fba_cache_append_rotary(c, k, v, x, xo, heads, r, None, None, None, tokens, t, out, None)
    append4 = lambda c=c4, k=q, x=None, xo=None, heads=0, r=None, tokens=1, t=0, out=out: lib.fba_cache4_append(c, k, q, x, xo, heads, r, None, None, None, tokens, t, out, None)
    attend = lambda c=c4, q=q, heads=4, window=99, sinks=0, acc=0, t=0, ws=f, n=1 << 40: lib.fba_cache4_attn(c, q, q, heads, window, sinks, acc, t, ws, n, None)
    evict = lambda c=c4, budget=8, recent=0, sinks=0, out=out, ws=f, n=1 << 40: lib.fba_cache4_evict(c, budget, recent, sinks, out, ws, n, None)
    read = lambda c=c4, first=0, slots=1, k=q, v=q, t=0: lib.fba_cache4_read(c, first, slots, k, v, t, None)
    read16 = lambda c=c, first=0, slots=1, k=q, t=0: lib.fba_cache_read(c, first, slots, k, q, t, None)
    for code, text, call in [
        (1, "head_dim", lambda: turn(D=64)), (1, "type", lambda: turn(t=2)), (1, "positive", lambda: turn(S=0)), (1, "positive", lambda: turn(Hq=0)), (1, "65535", lambda: turn(Hq=65536)),
        (1, "rotation is null", lambda: turn(r=None)), (1, "q is null", lambda: turn(q=None)), (1, "q_out is null", lambda: turn(o=None)), (1, "Hk", lambda: turn(k=q, ko=q)),
        (1, "Hk", lambda: turn(Hk=2)), (1, "k_out is null", lambda: turn(k=q, Hk=1)), (1, "strides", lambda: turn(q=odd)), (2, "2^27", lambda: turn(B=1 << 14, S=1 << 14)),
        (1, "cache is null", lambda: append(c=None)), (1, "rotation is null", lambda: append(r=None)), (1, "tokens", lambda: append(tokens=0)), (1, "type", lambda: append(t=-1)),
        (1, "k is null", lambda: append(k=None)), (1, "v: strides", lambda: append(v=odd)), (1, "heads", lambda: append(x=q, xo=q)), (1, "heads", lambda: append(heads=2)),
        (1, "q_out is null", lambda: append(x=q, heads=2)), (1, "lengths_out is null", lambda: append(out=None)), (1, "lengths_out must not", lambda: append(out=f)),
        (2, "2^27", lambda: append(tokens=1 << 26)), (2, "batch", lambda: append(c=ctypes.byref(Cache(**dict(GOOD, batch=(1 << 22) + 1))))),
        (1, "cache is null", lambda: append4(c=None)), (1, "k_scales", lambda: append4(c=_cache4(None))), (1, "k_scales", lambda: append4(c=_cache4(A + 4))), (1, "type", lambda: append4(t=2)),
        (1, "tokens", lambda: append4(tokens=0)), (1, "page_size", lambda: append4(c=_cache4(page_size=24))),
        (1, "cache is null", lambda: attend(c=None)), (1, "k_scales", lambda: attend(c=_cache4(None))), (1, "heads", lambda: attend(heads=3)), (1, "type", lambda: attend(t=2)),
        (1, "window", lambda: attend(window=0)), (1, "sinks", lambda: attend(sinks=-1)), (1, "whole cache", lambda: attend(acc=1, window=10)), (1, "weights is null", lambda: attend(_cache4(weights=None), acc=1)),
        (1, "ws must", lambda: attend(n=64)), (1, "ws must", lambda: attend(ws=None)), (1, "q is null", lambda: attend(q=None)), (2, "2^28", lambda: attend(_cache4(max_pages=1 << 25))),
        (1, "cache is null", lambda: evict(c=None)), (1, "k_scales", lambda: evict(c=_cache4(None))), (1, "budget", lambda: evict(budget=0)), (1, "fit the budget", lambda: evict(recent=9)),
        (1, "positions or weights", lambda: evict(_cache4(positions=None))), (1, "ws must", lambda: evict(n=4)), (1, "lengths_out is null", lambda: evict(out=None)),
        (1, "cache is null", lambda: read(c=None)), (1, "k_scales", lambda: read(c=_cache4(None))), (1, "first", lambda: read(first=-1)), (1, "slots", lambda: read(slots=0)),
        (1, "type", lambda: read(t=2)), (1, "v is null", lambda: read(v=None)), (1, "k: strides", lambda: read(k=odd)), (2, "launch", lambda: read(c=_cache4(batch=1 << 7, max_pages=1), slots=1 << 28)),
        (1, "cache is null", lambda: read16(c=None)), (1, "first", lambda: read16(first=(1 << 28) + 1)), (1, "slots", lambda: read16(slots=-1)), (1, "k is null", lambda: read16(k=None)),
    ]:
        assert call() == code, text
        assert text in lib.fba_last_error().decode(), lib.fba_last_error().decode()
    assert lib.fba_cache4_attn_workspace_bytes(None, 4, 0) == -1 and lib.fba_cache4_attn_workspace_bytes(c4, 3, 0) == -1 and lib.fba_cache4_attn_workspace_bytes(_cache4(None), 4, 0) == -1
    assert lib.fba_cache4_evict_workspace_bytes(None, 4) == -1 and lib.fba_cache4_evict_workspace_bytes(c4, 0) == -1
    assert lib.fba_cache4_attn_workspace_bytes(c4, 4, 1) - lib.fba_cache4_attn_workspace_bytes(c4, 4, 0) == 3 * 4 * 64 * 4
    assert lib.fba_cache4_evict_workspace_bytes(c4, 8) == lib.fba_cache_evict_workspace_bytes(c, 8)


def test_rotary_makes_turns_of_frequencies():
    import flex_block_attn_amd as fba

    r = fba.rotary((16, 56, 56), theta=256.0, device="cpu")
    assert (r.n_axes, r.interleaved, r.turns.dtype, r.axes.dtype) == (3, True, torch.int64, torch.int32)
    assert r.axes.tolist() == [0] * 8 + [1] * 28 + [2] * 28
    two_pi = Fraction(math.pi) * 2  # off by 2^-53 of itself, as are the frequencies
    for x, f in zip(r.turns.tolist(), [256.0 ** (-2 * j / d) for d in (16, 56, 56) for j in range(d // 2)]):
        want = Fraction(f) / two_pi * 2**64
        assert abs(x - want) <= want * 2.0**-51
    # several turns a step, and backwards: modulo whole turns
    r = fba.rotary((16,), frequencies=[2 * math.pi * 0.75, -2 * math.pi * 0.25, 2 * math.pi * 3.5, 0.0, 1.0, -1.0, 100.0, 1e-9], interleaved=False, device="cpu")
    assert r.turns.tolist()[:4] == [-(2**62), -(2**62), -(2**63), 0] and not r.interleaved
    assert r.turns[4] == -r.turns[5]
    r = fba.rotary((16,), frequencies=[1e300, -1e300, 2 * math.pi * 1e9, 0.0, 0.0, 0.0, 0.0, 0.0], device="cpu")  # as far as floats go
    assert r.turns[0] == -r.turns[1] and r.turns[2] == 0


@pytest.mark.parametrize("grid,tile", [((2, 4, 6), None), ((2, 4, 6), (1, 2, 3)), ((6, 8, 8), (6, 8, 8)), ((4, 4), (2, 4)), ((5,), None)])
def test_grid_coordinates(grid, tile):
    import flex_block_attn_amd as fba

    got = fba.grid_coordinates(grid, tile, device="cpu")
    every = [()]
    for n in grid:
        every = [(*x, i) for x in every for i in range(n)]
    if tile is not None:  # tiles in raster order, tokens of a tile in raster order
        every.sort(key=lambda x: ([a // t for a, t in zip(x, tile)], [a % t for a, t in zip(x, tile)]))
    assert got.dtype == torch.int32 and [tuple(x) for x in got.tolist()] == every


def test_python_refuses_without_a_gpu():
    import flex_block_attn_amd as fba

    z = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype)
    turn = fba.rotary(device="cpu")
    for dims in ((), (0,), (-2,), (3, 13), (8,), (128, 16), (16.0,), (True, 16), (2,) * 9):
        with pytest.raises(ValueError, match="dims"):
            fba.rotary(dims, device="cpu")
    for theta in (0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="theta"):
            fba.rotary(theta=theta, device="cpu")
    for frequencies in ([1.0] * 63, [math.nan] * 64, [math.inf] * 64):
        with pytest.raises(ValueError, match="frequencies"):
            fba.rotary(frequencies=frequencies, device="cpu")
    with pytest.raises(ValueError, match="whole tiles"):
        fba.grid_coordinates((2, 4, 6), (2, 3, 6), device="cpu")
    with pytest.raises(ValueError, match="GPU tensor"):
        fba.rotary_func(z(1, 1, 4, 128), None, turn)
    with pytest.raises(ValueError, match="bits"):
        fba.paged_cache(2, 1, bits=8, device="cpu")
    cache = fba.PagedCache4(z(2, 1, 16, 64, dtype=torch.uint8), z(2, 1, 16, 64, dtype=torch.uint8), z(2, 1, 16, 4, dtype=torch.uint8), z(2, 1, 16, 4, dtype=torch.uint8))
    table, n, k = z(1, 2, dtype=torch.int32), z(1, dtype=torch.int32), z(1, 1, 1, 128)
    for call in (lambda: fba.cache_append(cache, table, n, k, k), lambda: fba.cache_append_rotary(cache, table, n, k, k, turn), lambda: fba.cache_read(cache, table, n, 4),
                 lambda: fba.cache_attn_func(k, cache, table, n), lambda: fba.cache_evict(cache, table, n, 4)):
        with pytest.raises(ValueError, match="GPU tensor"):
            call()
    for call in (lambda: fba.cache_append_rotary(cache, table, n, k, k, None), lambda: fba.rotary_func(k, None, (turn.turns, turn.axes))):
        with pytest.raises((TypeError, ValueError), match="Rotary|GPU tensor"):
            call()
    with pytest.raises(TypeError, match="PagedCache"):
        fba.cache_read((cache.k, cache.v), table, n, 4)


@pytest.mark.gpu
def test_python_refuses_on_the_gpu(gpu):
    from dataclasses import replace

    import flex_block_attn_amd as fba
    from flex_block_attn_amd import _lib

    z = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype, device=gpu)
    i32, u8 = torch.int32, torch.uint8
    turn = fba.rotary((16, 56, 56), device=gpu)
    x, where = z(2, 3, 5, 128), z(5, 3, dtype=i32)
    f = fba.rotary_func
    for error, text, call in [
        (TypeError, "bfloat16 or float16", lambda: f(x.float(), None, turn)), (ValueError, "q's type", lambda: f(x, x.half(), turn)), (ValueError, "shape", lambda: f(x[0], None, turn)),
        (ValueError, "shape", lambda: f(x, x[:1], turn)), (ValueError, "shape", lambda: f(x, x[:, :, :4], turn)), (ValueError, "shape", lambda: f(x[..., :64], None, turn)),
        (ValueError, "GPU tensor", lambda: f(x, x.cpu(), turn)), (TypeError, "Rotary", lambda: f(x, None, turn.turns)),
        (ValueError, "turns", lambda: f(x, None, replace(turn, turns=turn.turns.int()))), (ValueError, "turns", lambda: f(x, None, replace(turn, turns=turn.turns.cpu()))),
        (ValueError, "axes", lambda: f(x, None, replace(turn, axes=turn.axes.long()))), (ValueError, "one length", lambda: f(x, None, replace(turn, axes=turn.axes[:8]))),
        (ValueError, "one length", lambda: f(x, None, replace(turn, turns=turn.turns[:12], axes=turn.axes[:12]))), (ValueError, "n_axes", lambda: f(x, None, replace(turn, n_axes=0))),
        (ValueError, "n_axes", lambda: f(x, None, replace(turn, n_axes=9))), (ValueError, "n_axes", lambda: f(x, None, replace(turn, n_axes=True))),
        (ValueError, "coordinates", lambda: f(x, None, turn, coordinates=where.long())), (ValueError, "coordinates", lambda: f(x, None, turn, coordinates=where[:4])),
        (ValueError, "coordinates", lambda: f(x, None, turn, coordinates=z(3, 5, 3, dtype=i32))), (ValueError, "coordinates", lambda: f(x, None, turn, coordinates=where.cpu())),
        (_lib.FbaError, "2\\^27", lambda: f(z(1, 1, 1, 128).expand(1 << 14, 1, 1 << 14, 128), None, turn)),
    ]:
        with pytest.raises(error, match=text):
            call()
    cache = fba.paged_cache(6, 2, 16, device=gpu, evicting=True, bits=4)
    plain = fba.PagedCache4(cache.k, cache.v, cache.k_scales, cache.v_scales)
    table, n, k, q = z(3, 2, dtype=i32), z(3, dtype=i32), z(3, 2, 5, 128), z(3, 4, 5, 128)
    one = fba.rotary(device=gpu)
    append, attend, read, evict = fba.cache_append_rotary, fba.cache_attn_func, fba.cache_read, fba.cache_evict
    for error, text, call in [
        (TypeError, "uint8", lambda: read(replace(cache, k=cache.k.view(torch.int8)), table, n, 4)), (TypeError, "dtype", lambda: read(replace(cache, dtype=torch.float32), table, n, 4)),
        (TypeError, "dtype", lambda: read(replace(cache, dtype=None), table, n, 4)), (ValueError, "shape", lambda: read(replace(cache, v=cache.v[:2]), table, n, 4)),
        (ValueError, "k_scales", lambda: read(replace(cache, k_scales=cache.k_scales[..., :2].contiguous()), table, n, 4)), (ValueError, "v_scales", lambda: read(replace(cache, v_scales=cache.v_scales[:, :, :, ::2]), table, n, 4)),
        (TypeError, "v_scales", lambda: read(replace(cache, v_scales=None), table, n, 4)), (ValueError, "GPU tensor", lambda: read(replace(cache, v_scales=cache.v_scales.cpu()), table, n, 4)),
        (ValueError, "aligned", lambda: read(replace(cache, k_scales=torch.zeros(cache.k_scales.numel() + 4, dtype=u8, device=gpu)[4:].view(cache.k_scales.shape)), table, n, 4)),
        (ValueError, "slots", lambda: read(cache, table, n, -1)), (TypeError, "slots", lambda: read(cache, table, n, 2.0)), (ValueError, "first", lambda: read(cache, table, n, 4, first=-1)),
        (_lib.FbaError, "2\\^28", lambda: read(cache, table, n, (1 << 28) + 1)),
        (TypeError, "k must have", lambda: append(cache, table, n, k.half(), k.half(), one)), (ValueError, "k and v must have shape", lambda: append(cache, table, n, k[:2], k[:2], one)),
        (TypeError, "q must have", lambda: append(cache, table, n, k, k, one, q=q.half())), (ValueError, "q must have shape", lambda: append(cache, table, n, k, k, one, q=q[:, :, :4])),
        (ValueError, "counts", lambda: append(cache, table, n, k, k, one, counts=n.long())), (ValueError, "positions", lambda: append(cache, table, n, k, k, one, positions=n[:1])),
        (ValueError, "coordinates", lambda: append(cache, table, n, k, k, turn, coordinates=z(4, 3, dtype=i32))), (ValueError, "has none", lambda: append(plain, table, n, k, k, one, weights=z(3, 2, 5, dtype=torch.float32))),
        (ValueError, "turns", lambda: append(cache, table, n, k, k, replace(one, turns=one.turns.cpu()))), (ValueError, "has none", lambda: fba.cache_append(plain, table, n, k, k, positions=n)),
        (ValueError, "no_grad", lambda: append(cache, table, n, k, k, one, q=q.clone().requires_grad_(True))), (ValueError, "no_grad", lambda: append(cache, table, n, k.clone().requires_grad_(True), k, one)),
        (TypeError, "q must have", lambda: attend(q[:, :, :1].half(), cache, table, n)), (ValueError, "q must have shape", lambda: attend(q, cache, table, n)),
        (ValueError, "with weights", lambda: attend(q[:, :, :1], plain, table, n, accumulate=True)), (ValueError, "window must be None", lambda: attend(q[:, :, :1], cache, table, n, window=4, accumulate=True)),
        (ValueError, "positions and weights", lambda: evict(plain, table, n, 4)), (ValueError, "budget", lambda: evict(cache, table, n, 0)),
        (_lib.FbaError, "2\\^27", lambda: append(cache, table, n, k[:, :, :1].expand(3, 2, 1 << 26, 128), k[:, :, :1].expand(3, 2, 1 << 26, 128), one)),
    ]:
        with pytest.raises(error, match=text):
            call()
    # nothing to do is no error
    out, none = append(cache, table, n, k[:, :, :0], k[:, :, :0], one, q=q[:, :, :0])
    assert out.tolist() == [0, 0, 0] and none.shape == (3, 4, 0, 128)
    assert [t.shape for t in read(cache, table, n, 0)] == [(3, 2, 0, 128)] * 2
    for e in (x[:, :, :0], x[:0], x[:, :0]):
        assert f(e, None, turn)[0].shape == e.shape
    assert [t.shape for t in f(x[:, :0], x, turn)] == [(2, 0, 5, 128), (2, 3, 5, 128)]
