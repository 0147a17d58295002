"""Positions by rotation, on one axis (text) or several (time, height and width of a video's tokens): q and k are turned, pair by pair, by angles that grow with where their tokens
stand, before they go to `window_attn_func`, `ssta_3d_attention` or a paged cache (`cache_append_rotary` turns them on the way).  The kernel is csrc/fba_rotary.hip; what it computes is
stated in include/fba.h.

    turn = rotary((16, 56, 56))                                        # once: columns of time, height and width, 128 together
    where = grid_coordinates((T, H, W))                                # once for a grid: (T * H * W, 3)
    q, k = rotary_func(q, k, turn, coordinates=where)                  # (batch, heads, seq, 128), differentiable
"""
import math
import numbers
from dataclasses import dataclass

import torch

from . import _lib
from .interface import HEAD_DIM, _require_device, _typed_like
from .window import _TYPES, _rows_dense


@dataclass(frozen=True)
class Rotary:
    """What the pairs of a row turn by; made by `rotary`.  Pair i is the columns (2i, 2i + 1) if interleaved, else (i, i + pairs); what is behind the pairs stays as it is."""

    turns: torch.Tensor  # (pairs,) int64: turns of one step, times 2^64, modulo 2^64; pairs a multiple of 8, 64 at most
    axes: torch.Tensor   # (pairs,) int32: the axis whose steps count; one that is not below n_axes counts as the last
    n_axes: int = 1      # 8 at most
    interleaved: bool = True


def rotary(dims=(HEAD_DIM,), theta=10000.0, interleaved=True, frequencies=None, device="cuda"):
    """dims: how many columns every axis has, even numbers whose sum is a multiple of 16, 128 at most.  The j-th pair of an axis of d columns turns by theta^(-2j / d) radians a
    step; `frequencies`, one number for every pair, axis by axis, replaces that (scaled or shared spectra).

    Both are worked out in doubles, and so are the turns of a step, frequency / (2 pi): 2^-52 of the step off at most, and 2^-64 of a turn.  At a coordinate c, an angle is off by
    2^-52 |c| frequency radians therefore (5e-7 at 2^31, for a frequency of one).  Who needs more makes a `Rotary` of turns of their own."""
    dims = tuple(dims)
    if not dims or len(dims) > 8 or not all(isinstance(d, numbers.Integral) and not isinstance(d, bool) and d > 0 and d % 2 == 0 for d in dims):
        raise ValueError(f"dims must be one to eight positive even numbers, got {dims}")
    if sum(dims) % 16 or sum(dims) > HEAD_DIM:
        raise ValueError(f"the sum of dims ({sum(dims)}) must be a multiple of 16, {HEAD_DIM} at most")
    if frequencies is None:
        if not 0 < theta < math.inf:
            raise ValueError(f"theta ({theta}) must be a positive number")
        frequencies = [theta ** (-2 * j / d) for d in dims for j in range(d // 2)]
    frequencies = [float(f) for f in frequencies]
    if len(frequencies) != sum(dims) // 2 or not all(map(math.isfinite, frequencies)):
        raise ValueError(f"frequencies must be {sum(dims) // 2} finite numbers, got {len(frequencies)}")
    turns = [(int(math.fmod(f / (2 * math.pi), 1.0) * 2**64) + 2**63) % 2**64 - 2**63 for f in frequencies]  # (the quotient is off by 2^-53 of itself, and 2^-54.5 for that pi; whole turns off, times a power of two: both exact)
    turns, axes = torch.tensor(turns, dtype=torch.int64), torch.tensor([x for x, d in enumerate(dims) for _ in range(d // 2)], dtype=torch.int32)
    return Rotary(turns.to(device), axes.to(device), len(dims), bool(interleaved))


def grid_coordinates(grid, tile=None, device="cuda"):
    """Where the tokens of a grid (T, H, W) stand: int32 (T * H * W, 3), in raster order or, with `tile`, in that of `tile_tokens`."""
    grid = tuple(grid)
    where = torch.stack(torch.meshgrid(*(torch.arange(n, dtype=torch.int32) for n in grid), indexing="ij"), -1)
    if tile is not None:
        tile = tuple(tile)
        if len(tile) != len(grid) or any(t <= 0 or n % t for n, t in zip(grid, tile)):
            raise ValueError(f"grid {grid} must be whole tiles of {tile}")
        n = len(grid)
        cut = [x for size, t in zip(grid, tile) for x in (size // t, t)]
        where = where.reshape(*cut, n).permute(*range(0, 2 * n, 2), *range(1, 2 * n, 2), 2 * n)
    return where.reshape(-1, len(grid)).contiguous().to(device)


def _check_rotary(rotary, like):
    if not isinstance(rotary, Rotary):
        raise TypeError(f"rotary must be a Rotary, got {type(rotary).__name__}")
    turns, axes = rotary.turns, rotary.axes
    for name, t, dtype in (("turns", turns, torch.int64), ("axes", axes, torch.int32)):
        if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != 1 or t.device != like.device or not t.is_contiguous():
            raise ValueError(f"rotary.{name} must be {dtype} of shape (pairs,) on {like.device}, contiguous")
    if turns.shape != axes.shape or not 8 <= turns.shape[0] <= HEAD_DIM // 2 or turns.shape[0] % 8:
        raise ValueError(f"rotary.turns and rotary.axes must have one length, a multiple of 8 and {HEAD_DIM // 2} at most, got {turns.shape[0]} and {axes.shape[0]}")
    if isinstance(rotary.n_axes, bool) or not isinstance(rotary.n_axes, numbers.Integral) or not 1 <= rotary.n_axes <= 8:
        raise ValueError(f"rotary.n_axes ({rotary.n_axes}) must be an integer between 1 and 8")


def _check_coordinates(coordinates, rotary, batch, tokens, like):
    if coordinates is None:
        return None
    shapes = ((tokens, rotary.n_axes), (batch, tokens, rotary.n_axes))
    if not isinstance(coordinates, torch.Tensor) or coordinates.dtype != torch.int32 or coordinates.device != like.device or tuple(coordinates.shape) not in shapes:
        raise ValueError(f"coordinates must be int32 of shape {shapes[0]} or {shapes[1]} on {like.device}")
    return coordinates.contiguous()


def _check_rotary_args(q, k, rotary, coordinates):
    """Raises for everything that the kernel does not take.  -> coordinates, dense"""
    for name, t in (("q", q), ("k", k)):
        if name == "k" and t is None:
            continue
        _require_device(t, name)
        if t.dtype not in _TYPES:
            raise TypeError(f"{name} must be bfloat16 or float16, got {t.dtype}")
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{name} must have q's type and device ({q.dtype}, {q.device}), got {t.dtype}, {t.device}")
        if t.dim() != 4 or t.shape[3] != HEAD_DIM or t.shape[0] != q.shape[0] or t.shape[2] != q.shape[2] or t.shape[1] > 65535:
            raise ValueError(f"{name} must have shape (batch, heads, seq, {HEAD_DIM}), batch and seq those of q, 65535 heads at most, got {tuple(t.shape)}")
    _check_rotary(rotary, q)
    if q.shape[0] * q.shape[2] > 1 << 27:
        raise _lib.FbaError(_lib.FBA_ERR_UNSUPPORTED, f"all sequences together may have 2^27 tokens, got {q.shape[0]} x {q.shape[2]}")
    return _check_coordinates(coordinates, rotary, q.shape[0], q.shape[2], q)


class RotaryFunc(torch.autograd.Function):
    """The operator as a Python autograd function: for arguments that need preparation or are refused, calls that are traced and tensor subclasses."""

    @staticmethod
    def forward(ctx, q, k, turns, axes, n_axes, interleaved, coordinates, inverse):
        coordinates = _check_rotary_args(q, k, Rotary(turns, axes, n_axes, interleaved), coordinates)
        n_axes, interleaved, inverse = int(n_axes), bool(interleaved), bool(inverse)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(turns, axes, coordinates)
        ctx.args = (n_axes, interleaved, inverse)
        q, k = _rows_dense(q), None if k is None else _rows_dense(k)
        out_q, out_k = _lib.host().rotary_forward(q, k, turns, axes, n_axes, interleaved, coordinates, inverse)
        return _typed_like(out_q, q), None if out_k is None else _typed_like(out_k, k)

    @staticmethod
    def backward(ctx, gq, gk):
        turns, axes, coordinates = ctx.saved_tensors
        n_axes, interleaved, inverse = ctx.args
        gq, gk = (g if need else None for g, need in zip((gq, gk), ctx.needs_input_grad))
        if gq is None and gk is None:
            return (None,) * 8
        if gq is None:
            gk, _ = RotaryFunc.apply(gk, None, turns, axes, n_axes, interleaved, coordinates, not inverse)
        else:
            gq, gk = RotaryFunc.apply(gq, gk, turns, axes, n_axes, interleaved, coordinates, not inverse)
        return (gq, gk) + (None,) * 6


def rotary_func(q, k, rotary, coordinates=None, inverse=False):
    """q (batch, heads, seq, 128) and k (batch, kv_heads, seq, 128; None: q alone) with every row's pairs turned by where its token stands: (a, b) -> (a cos w - b sin w, a sin w + b cos w),
    w = frequency * coordinate on the pair's axis.

    bf16 or fp16, any strides with dense rows.  coordinates: int32 (seq, n_axes) or (batch, seq, n_axes) on the GPU, any values; None: row t stands at t on every axis.  The angle of any
    coordinate is the multiple of a step's turns, `rotary.turns`, modulo whole turns, without rounding (how near these are to the frequencies: `rotary`); sines, cosines and products are fp32,
    the result is rounded once.  Rows of padding are turned too.  inverse: turned back.

    Returns (q, k), new tensors, k None if it was.  Differentiable in q and k, as often as wanted; coordinates and rotary must not be written to before backward has come.  A step may be
    captured into a graph, under the condition that `window_attn_func` states."""
    of = (rotary.turns, rotary.axes, rotary.n_axes, rotary.interleaved) if isinstance(rotary, Rotary) else None
    out = None if of is None else _lib.host().rotary(q, k, *of, coordinates, bool(inverse))
    if out is not None:
        return out
    if of is None:
        raise TypeError(f"rotary must be a Rotary, got {type(rotary).__name__}")
    return RotaryFunc.apply(q, k, *of, coordinates, inverse)
