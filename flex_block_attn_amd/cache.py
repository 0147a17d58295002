"""A paged cache of keys and values for streams of tokens, the attention of single new tokens over it, and eviction by accumulated attention weight: what serves a
model that was trained with `window_attn_func` or plain causal attention.  The kernels are csrc/fba_cache.hip and csrc/fba_cache_attend.hip; what they do is stated
in include/fba.h.

A step of a batch of sequences, which may be captured into a graph:

    cache = paged_cache(pages, kv_heads, page_size, evicting=True)
    lengths = cache_append(cache, table, lengths, k, v, positions=seen)       # the new token's rows
    o = cache_attn_func(q, cache, table, lengths, accumulate=True)            # what it reads, and what that weighed
    lengths = cache_evict(cache, table, lengths, budget, recent=256, sinks=4)

`table`, int32 (batch, max_pages): the pages of every sequence, in order; which pages are free is the caller's to keep.  `lengths`, int32 (batch,): filled slots.  Both
are read on the GPU: a length that is negative or beyond the table, or a page outside of the pool, answers NaN or a length of -1 for that sequence.  A page that a call
writes to may be in one place of the table only.

Weights come from `cache_attn_func(accumulate=True)`, or from the caller: a prompt's rows have those that `cache_append` is given, zeros otherwise (`window_attn_func` leaves none).  An
eviction right after a prompt without any goes by `sinks`, `recent` and, among equals, the lower slot.

Keys that carry their positions by rotation (positions.py) are turned on the way in, and the step's q beside them:

    lengths, q = cache_append_rotary(cache, table, lengths, k, v, turn, q=q)

A prompt's next chunk sees what is cached through `cache_read`, which hands rows back as dense tensors, for `window_attn_func`:

    lengths, q = cache_append_rotary(cache, table, lengths, k, v, turn, q=q, counts=counts)
    o = window_attn_func(q, *cache_read(cache, table, lengths, before + tokens), window)

`window_attn_func` takes the queries for the last rows that it is given, of all sequences alike.  So this is for sequences that had one length, `before`, in front of the chunk; counts may
differ (o behind a sequence's count is of nothing).  Where `before` differs the queries of a shorter sequence would stand behind its end, and see rows of zeros and tokens that come after
them: such sequences go one by one, each with table[b:b + 1], lengths[b:b + 1], as many slots as it has, and its own queries.

The pool may hold 4 bits to a value instead of 16 (`paged_cache(bits=4)`): 136 bytes instead of 512 for a slot's key and value.  All calls take either; attention is then over what the 4
bits stand for, which is exact in the pool's type.  The kernels are csrc/fba_cache_rotary.hip and csrc/fba_cache_attend4.hip.

What a call writes to counts as changed in place: a backward pass that has saved it raises.
"""
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .interface import HEAD_DIM, _require_device
from .positions import Rotary, _check_coordinates, _check_rotary
from .window import _NO_WINDOW, _TYPES, _rows_dense, _whole


@dataclass
class PagedCache:
    """The pool of pages.  `positions` (where in its sequence a slot's token stood) and `weights` (what attention has given it so far) go with the slots of every kv head;
    eviction needs both, append fills what there is."""

    k: torch.Tensor  # (pages, kv_heads, page_size, 128) bf16 or fp16, contiguous; page_size a power of two, 16 at least
    v: torch.Tensor
    positions: Optional[torch.Tensor] = None  # (pages, kv_heads, page_size) int32
    weights: Optional[torch.Tensor] = None    # (pages, kv_heads, page_size) float32


@dataclass
class PagedCache4:
    """The pool of pages in 4 bits: value 2j of a row in the low half of byte j, 2j + 1 in the high one, 0, 0.5, 1, 1.5, 2, 3, 4 or 6 with a sign (the fourth bit), times 2^(scale - 127),
    a scale for every 32 values; 255: they are no numbers.  What is appended goes to the nearest, ties to the even code; 2^(scale - 127) is a quarter of the power of two below the
    largest of the 32, or a half from 1.75 times that power on.  So a value v is off by a quarter of 2^(scale - 127) or of |v| at most (and what is beyond 7 * 2^125, in fp16 7 * 2^13,
    becomes 6 * 2^125, 6 * 2^13); an infinity takes its 32 with it."""

    k: torch.Tensor  # (pages, kv_heads, page_size, 64) uint8, contiguous; page_size a power of two, 16 at least
    v: torch.Tensor
    k_scales: torch.Tensor  # (pages, kv_heads, page_size, 4) uint8
    v_scales: torch.Tensor
    dtype: torch.dtype = torch.bfloat16       # of what it stands for, and of q, k, v and o; fixed for a pool
    positions: Optional[torch.Tensor] = None  # (pages, kv_heads, page_size) int32
    weights: Optional[torch.Tensor] = None    # (pages, kv_heads, page_size) float32


def paged_cache(pages, kv_heads, page_size=64, dtype=torch.bfloat16, device="cuda", evicting=False, bits=16):
    """An empty pool, with positions and weights if it is to be evicted from: a PagedCache, or with bits=4 a PagedCache4.  Its memory is not initialised: no call reads a slot that was
    not filled."""
    page_size = _page_size(_whole(page_size, "page_size", 16))
    pages, kv_heads = _whole(pages, "pages", 1), _whole(kv_heads, "kv_heads", 1)
    if dtype not in _TYPES:
        raise TypeError(f"dtype must be bfloat16 or float16, got {dtype}")
    if bits not in (4, 16):
        raise ValueError(f"bits must be 4 or 16, got {bits}")
    pool = (pages, kv_heads, page_size)
    rows = lambda n, of: [torch.empty((*pool, n), dtype=of, device=device) for _ in range(2)]
    k, v = rows(HEAD_DIM, dtype) if bits == 16 else rows(HEAD_DIM // 2, torch.uint8)
    _require_device(k, "the cache")
    slots = (torch.empty(pool, dtype=torch.int32, device=device), torch.empty(pool, dtype=torch.float32, device=device)) if evicting else ()
    return PagedCache(k, v, *slots) if bits == 16 else PagedCache4(k, v, *rows(HEAD_DIM // 32, torch.uint8), dtype, *slots)


def _page_size(n):
    if n < 16 or n & (n - 1):
        raise ValueError(f"page_size ({n}) must be a power of two, 16 at least")
    return n


def _given(cache, table, lengths, positions=True):
    """The tensors of a call as the native side takes them, and the type of the cache's values; None for what is no cache.  positions=False: a call that has no use for the cache's."""
    if isinstance(cache, PagedCache):
        return (cache.k, cache.v, None, None, cache.positions if positions else None, cache.weights, table, lengths, getattr(cache.k, "dtype", None))
    if isinstance(cache, PagedCache4):
        return (cache.k, cache.v, cache.k_scales, cache.v_scales, cache.positions if positions else None, cache.weights, table, lengths, cache.dtype)
    return None


def _check_cache(cache, table, lengths, positions=True):
    """Raises for everything that the kernels do not take; positions=False: of a call that has no use for the cache's.  -> the type of the cache's values"""
    if not isinstance(cache, (PagedCache, PagedCache4)):
        raise TypeError(f"cache must be a PagedCache or a PagedCache4, got {type(cache).__name__}")
    k, held = cache.k, isinstance(cache, PagedCache4)
    own = cache.positions if positions else None
    tensors = [("k", k), ("v", cache.v), ("positions", own), ("weights", cache.weights)]
    if held:
        tensors += [("k_scales", cache.k_scales), ("v_scales", cache.v_scales)]
    tensors = [("cache." + name, t) for name, t in tensors if t is not None or name not in ("positions", "weights")]
    for name, t in (*tensors, ("table", table), ("lengths", lengths)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
        _require_device(t, name)
        if t.device != k.device:
            raise ValueError(f"{name} must be on the cache's device ({k.device}), got {t.device}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    if held:
        if cache.dtype not in _TYPES:
            raise TypeError(f"cache.dtype must be bfloat16 or float16, got {cache.dtype}")
        if any(t.dtype != torch.uint8 for t in (k, cache.v, cache.k_scales, cache.v_scales)):
            raise TypeError("cache.k, cache.v, cache.k_scales and cache.v_scales must be uint8")
    elif k.dtype not in _TYPES or cache.v.dtype != k.dtype:
        raise TypeError(f"cache.k and cache.v must both be bfloat16 or float16, got {k.dtype} and {cache.v.dtype}")
    width = HEAD_DIM // 2 if held else HEAD_DIM
    if k.dim() != 4 or k.shape[3] != width or cache.v.shape != k.shape:
        raise ValueError(f"cache.k and cache.v must have shape (pages, kv_heads, page_size, {width}), got {tuple(k.shape)} and {tuple(cache.v.shape)}")
    _page_size(k.shape[2])
    if k.numel() == 0:
        raise ValueError(f"the cache must have a page and a head, got {tuple(k.shape)}")
    if held and any(t.shape != (*k.shape[:3], HEAD_DIM // 32) for t in (cache.k_scales, cache.v_scales)):
        raise ValueError(f"cache.k_scales and cache.v_scales must have shape {(*k.shape[:3], HEAD_DIM // 32)}, got {tuple(cache.k_scales.shape)} and {tuple(cache.v_scales.shape)}")
    for name, t, dtype in (("positions", own, torch.int32), ("weights", cache.weights, torch.float32)):
        if t is not None and (t.dtype != dtype or t.shape != k.shape[:3]):
            raise ValueError(f"cache.{name} must be {dtype} of shape {tuple(k.shape[:3])}, got {t.dtype} {tuple(t.shape)}")
    if table.dtype != torch.int32 or table.dim() != 2 or table.numel() == 0:
        raise ValueError(f"table must be int32 of shape (batch, max_pages), not empty, got {table.dtype} {tuple(table.shape)}")
    if lengths.dtype != torch.int32 or tuple(lengths.shape) != (table.shape[0],):
        raise ValueError(f"lengths must be int32 of shape ({table.shape[0]},), got {lengths.dtype} {tuple(lengths.shape)}")
    if table.shape[1] * k.shape[2] > 1 << 28 or table.shape[0] > 0x7fffff or k.shape[1] > 65535 or k.shape[0] > 0x7fffffff:
        raise _lib.FbaError(_lib.FBA_ERR_UNSUPPORTED, f"a sequence may have 2^28 slots at most, a pool 2^31 - 1 pages of 65535 heads, got table {tuple(table.shape)}, cache {tuple(k.shape)}")
    for name, t in tensors:
        if t.data_ptr() % 16:
            raise ValueError(f"{name} must be 16-byte aligned")
    return cache.dtype if held else k.dtype


def _check_ints(t, name, table):
    if t is not None and (not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or tuple(t.shape) != (table.shape[0],) or t.device != table.device):
        raise ValueError(f"{name} must be int32 of shape ({table.shape[0]},) on {table.device}")


def _no_gradients(**tensors):
    if torch.is_grad_enabled():
        for name, t in tensors.items():
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} requires gradients: the cache's operators have no backward pass, call them under torch.no_grad()")


def _answered(result):
    if result is None:  # (a subclass of Tensor, a transformed call)
        raise TypeError("the cache's operators take plain tensors, outside of traces and function transforms")
    return result


def _check_rows(table, kv_heads, like, dtype, k, v):
    batch = table.shape[0]
    for name, t in (("k", k), ("v", v)):
        _require_device(t, name)
        if t.dtype != dtype or t.device != like.device:
            raise TypeError(f"{name} must have the cache's type and device ({dtype}, {like.device}), got {t.dtype}, {t.device}")
        if t.dim() != 4 or t.shape[0] != batch or t.shape[1] != kv_heads or t.shape[3] != HEAD_DIM or t.shape != k.shape:
            raise ValueError(f"k and v must have shape ({batch}, {kv_heads}, tokens, {HEAD_DIM}), got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.shape[2] > 1 << 28:
        raise _lib.FbaError(_lib.FBA_ERR_UNSUPPORTED, f"a call may append 2^28 tokens at most, got {k.shape[2]}")


def _append(cache, table, lengths, k, v, counts, positions, weights, q=None, rotary=None, coordinates=None):
    """-> (lengths, q turned)"""
    given = _given(cache, table, lengths)
    turn = (None, None, None, None) if rotary is None else (rotary.turns, rotary.axes, rotary.n_axes, rotary.interleaved) if isinstance(rotary, Rotary) else None
    out = None if given is None or turn is None else _lib.host().cache_append(given, k, v, counts, positions, weights, q, *turn, coordinates)
    if out is not None:
        return out
    dtype = _check_cache(cache, table, lengths)
    _check_rows(table, cache.k.shape[1], cache.k, dtype, k, v)
    batch, tokens = k.shape[0], k.shape[2]
    _check_ints(counts, "counts", table)
    _check_ints(positions, "positions", table)
    if positions is not None and cache.positions is None and rotary is None:
        raise ValueError("positions are given, but the cache has none")
    if weights is not None:
        if cache.weights is None:
            raise ValueError("weights are given, but the cache has none")
        if weights.dtype != torch.float32 or weights.shape != k.shape[:3] or weights.device != k.device:
            raise ValueError(f"weights must be float32 of shape {tuple(k.shape[:3])} on {k.device}, got {weights.dtype} {tuple(weights.shape)} on {weights.device}")
    if rotary is not None:
        _check_rotary(rotary, k)
        coordinates = _check_coordinates(coordinates, rotary, batch, tokens, k)
    if q is not None:
        _require_device(q, "q")
        if q.dtype != dtype or q.device != k.device:
            raise TypeError(f"q must have the cache's type and device ({dtype}, {k.device}), got {q.dtype}, {q.device}")
        if q.dim() != 4 or q.shape[0] != batch or q.shape[2] != tokens or q.shape[3] != HEAD_DIM or not 1 <= q.shape[1] <= 65535:
            raise ValueError(f"q must have shape ({batch}, heads, {tokens}, {HEAD_DIM}), 65535 heads at most, got {tuple(q.shape)}")
    if (rotary is not None or isinstance(cache, PagedCache4)) and (batch * tokens > 1 << 27 or batch > 1 << 22):
        raise _lib.FbaError(_lib.FBA_ERR_UNSUPPORTED, f"all sequences together may have 2^27 new tokens, and a batch 2^22 of them, got {batch} x {tokens}")
    _no_gradients(**{"cache.k": cache.k, "cache.v": cache.v, "cache.weights": cache.weights, "k": k, "v": v, "weights": weights, "q": q})
    if tokens == 0:
        right = (lengths >= 0) & (lengths <= table.shape[1] * cache.k.shape[2])
        return torch.where(right if counts is None else right & (counts == 0), lengths, -1), None if q is None else torch.empty_like(q)
    dense = lambda t: None if t is None else t.contiguous()
    rows = lambda t: None if t is None else _rows_dense(t)
    if rotary is not None:
        turn = (*turn[:2], int(rotary.n_axes), bool(rotary.interleaved))
    return _answered(_lib.host().cache_append(given, rows(k), rows(v), dense(counts), dense(positions), dense(weights), rows(q), *turn, coordinates))


def cache_append(cache, table, lengths, k, v, counts=None, positions=None, weights=None):
    """Rows of new tokens go to the slots behind `lengths`: k, v (batch, kv_heads, tokens, 128), any strides with dense rows; of sequence b the first counts[b] (int32
    (batch,); None: all).  Where the cache has positions, the tokens' are positions[b], positions[b] + 1, ... (int32 (batch,); None: those of the slots, right
    as long as nothing has been evicted); where it has weights, they begin with `weights` (float32 (batch, kv_heads, tokens); None: zero).

    Returns the new lengths, a tensor of its own: lengths + counts, and -1 where length or count make no sense, there is no room (nothing is written then) or a page is
    outside of the pool (its rows are not written)."""
    return _append(cache, table, lengths, k, v, counts, positions, weights)[0]


def cache_append_rotary(cache, table, lengths, k, v, rotary, q=None, counts=None, positions=None, weights=None, coordinates=None):
    """`cache_append` with k turned by `rotary` (positions.py) on the way, and q (batch, heads, tokens, 128), if given, beside it; in one launch.  The tokens of sequence b stand at
    positions[b], positions[b] + 1, ... on every axis (None: at their slots; a cache without positions takes them too), or at `coordinates`, int32 (tokens, n_axes) or
    (batch, tokens, n_axes), which the cache's own positions do not follow.  A k that goes into 4 bits is rounded once.

    Returns the new lengths, as `cache_append` does, and q turned (None without): its rows behind a sequence's count too, and no numbers for a sequence whose length or count makes no
    sense or that has no room (but q turned where only a page is outside of the pool)."""
    if not isinstance(rotary, Rotary):
        raise TypeError(f"rotary must be a Rotary, got {type(rotary).__name__}")
    return _append(cache, table, lengths, k, v, counts, positions, weights, q, rotary, coordinates)


def cache_read(cache, table, lengths, slots, first=0):
    """Slots first .. first + slots - 1 of every sequence as dense tensors k, v (batch, kv_heads, slots, 128) of the cache's type: what a prompt's next chunk attends to with
    `window_attn_func`, where all sequences had one length in front of it (else one by one: the head of this file).  Rows behind a sequence's length are zeros; those of a page outside of the pool, and all of a sequence whose length makes no sense, are no numbers."""
    given = _given(cache, table, lengths)
    out = None if given is None else _lib.host().cache_read(given, slots, first)
    if out is not None:
        return out
    dtype = _check_cache(cache, table, lengths)
    slots, first = _whole(slots, "slots", 0), _whole(first, "first", 0)
    if slots > 1 << 28 or first > 1 << 28:
        raise _lib.FbaError(_lib.FBA_ERR_UNSUPPORTED, f"a sequence has 2^28 slots at most, got first {first} and slots {slots}")
    _no_gradients(**{"cache.k": cache.k, "cache.v": cache.v})
    if slots == 0:
        return tuple(torch.empty((table.shape[0], cache.k.shape[1], 0, HEAD_DIM), dtype=dtype, device=cache.k.device) for _ in range(2))
    return _answered(_lib.host().cache_read(given, slots, first))


def cache_attn_func(q, cache, table, lengths, window=None, sinks=0, accumulate=False):
    """Attention of one new token per sequence, the last of its `lengths` slots: softmax(q k^T / sqrt(128)) v over the filled slots or, with `window`, over the last
    `window` of them and the first `sinks`.  (Slots are in the order of tokens as long as nothing has been evicted.)

    q: (batch, heads, 1, 128) of the cache's type, heads a multiple of kv_heads.  accumulate=True adds to cache.weights what softmax gave every slot, summed over the query
    heads of a kv head; not with a window, and with a workspace of 4 * batch * heads bytes for every slot that the table has room for, filled or not.  The cache's positions are not looked at.  Returns o, shaped like q: zeros for a sequence without slots, NaN for one whose length or pages make no sense."""
    given = _given(cache, table, lengths, positions=False)
    out = None if given is None else _lib.host().cache_attention(q, given, window, sinks, bool(accumulate))
    if out is not None:
        return out
    dtype = _check_cache(cache, table, lengths, positions=False)
    _require_device(q, "q")
    if q.dtype != dtype or q.device != cache.k.device:
        raise TypeError(f"q must have the cache's type and device ({dtype}, {cache.k.device}), got {q.dtype}, {q.device}")
    if q.dim() != 4 or q.shape[0] != table.shape[0] or q.shape[2] != 1 or q.shape[3] != HEAD_DIM:
        raise ValueError(f"q must have shape ({table.shape[0]}, heads, 1, {HEAD_DIM}), got {tuple(q.shape)}")
    if q.shape[1] == 0 or q.shape[1] % cache.k.shape[1] or q.shape[1] > 65535:
        raise ValueError(f"q heads ({q.shape[1]}) must be a multiple of the cache's ({cache.k.shape[1]}), 65535 at most")
    if accumulate and cache.weights is None:
        raise ValueError("accumulate needs a cache with weights")
    if accumulate and window is not None:
        raise ValueError("weights are added up over the whole cache: window must be None")
    window = _NO_WINDOW if window is None else _whole(window, "window", 1)
    sinks = _whole(sinks, "sinks", 0)
    _no_gradients(**{"q": q, "cache.k": cache.k, "cache.v": cache.v, "cache.weights": cache.weights})
    return _answered(_lib.host().cache_attention(_rows_dense(q), given, None if window == _NO_WINDOW else window, sinks, bool(accumulate)))


def cache_evict(cache, table, lengths, budget, recent=0, sinks=0):
    """Brings every sequence of more than `budget` slots down to that, every kv head for itself: tokens at positions below `sinks` and the `recent` last ones stay, then those
    with the largest weights (of equal ones the lower slot; NaN is the lowest).  Slots that are freed below the budget take the kept ones from behind it, in order: rows,
    positions and weights; slots are in no order of tokens then.  batch * kv_heads may be 65535 at most.

    Returns the new lengths, a tensor of its own: min(lengths, budget), and -1, with nothing moved, where a length or page makes no sense."""
    given = _given(cache, table, lengths)
    out = None if given is None else _lib.host().cache_evict(given, budget, recent, sinks)
    if out is not None:
        return out
    _check_cache(cache, table, lengths)
    if cache.positions is None or cache.weights is None:
        raise ValueError("eviction needs a cache with positions and weights")
    budget, recent, sinks = _whole(budget, "budget", 1), _whole(recent, "recent", 0), _whole(sinks, "sinks", 0)
    if recent + sinks > budget:
        raise ValueError(f"recent ({recent}) and sinks ({sinks}) must fit the budget ({budget}) together")
    _no_gradients(**{"cache.k": cache.k, "cache.v": cache.v, "cache.weights": cache.weights})
    return _answered(_lib.host().cache_evict(given, budget, recent, sinks))
