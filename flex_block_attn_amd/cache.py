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

What a call writes to counts as changed in place: a backward pass that has saved it raises.
"""
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .interface import HEAD_DIM, _require_device
from .window import _NO_WINDOW, _TYPES, _rows_dense, _whole


@dataclass
class PagedCache:
    """The pool of pages.  `positions` (where in its sequence a slot's token stood) and `weights` (what attention has given it so far) go with the slots of every kv head;
    eviction needs both, append fills what there is."""

    k: torch.Tensor  # (pages, kv_heads, page_size, 128) bf16 or fp16, contiguous; page_size a power of two, 16 at least
    v: torch.Tensor
    positions: Optional[torch.Tensor] = None  # (pages, kv_heads, page_size) int32
    weights: Optional[torch.Tensor] = None    # (pages, kv_heads, page_size) float32


def paged_cache(pages, kv_heads, page_size=64, dtype=torch.bfloat16, device="cuda", evicting=False):
    """An empty pool, with positions and weights if it is to be evicted from.  Its memory is not initialised: no call reads a slot that was not filled."""
    page_size = _page_size(_whole(page_size, "page_size", 16))
    pages, kv_heads = _whole(pages, "pages", 1), _whole(kv_heads, "kv_heads", 1)
    if dtype not in _TYPES:
        raise TypeError(f"dtype must be bfloat16 or float16, got {dtype}")
    k, v = (torch.empty((pages, kv_heads, page_size, HEAD_DIM), dtype=dtype, device=device) for _ in range(2))
    _require_device(k, "the cache")
    if not evicting:
        return PagedCache(k, v)
    return PagedCache(k, v, torch.empty(k.shape[:3], dtype=torch.int32, device=device), torch.empty(k.shape[:3], dtype=torch.float32, device=device))


def _page_size(n):
    if n < 16 or n & (n - 1):
        raise ValueError(f"page_size ({n}) must be a power of two, 16 at least")
    return n


def _check_cache(cache, table, lengths):
    """Raises for everything that the kernels do not take."""
    if not isinstance(cache, PagedCache):
        raise TypeError(f"cache must be a PagedCache, got {type(cache).__name__}")
    k = cache.k
    for name, t in (("cache.k", k), ("cache.v", cache.v), ("cache.positions", cache.positions), ("cache.weights", cache.weights), ("table", table), ("lengths", lengths)):
        if t is None and name in ("cache.positions", "cache.weights"):
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
        _require_device(t, name)
        if t.device != k.device:
            raise ValueError(f"{name} must be on the cache's device ({k.device}), got {t.device}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    if k.dtype not in _TYPES or cache.v.dtype != k.dtype:
        raise TypeError(f"cache.k and cache.v must both be bfloat16 or float16, got {k.dtype} and {cache.v.dtype}")
    if k.dim() != 4 or k.shape[3] != HEAD_DIM or cache.v.shape != k.shape:
        raise ValueError(f"cache.k and cache.v must have shape (pages, kv_heads, page_size, {HEAD_DIM}), got {tuple(k.shape)} and {tuple(cache.v.shape)}")
    _page_size(k.shape[2])
    if k.numel() == 0:
        raise ValueError(f"the cache must have a page and a head, got {tuple(k.shape)}")
    for name, t, dtype in (("positions", cache.positions, torch.int32), ("weights", cache.weights, torch.float32)):
        if t is not None and (t.dtype != dtype or t.shape != k.shape[:3]):
            raise ValueError(f"cache.{name} must be {dtype} of shape {tuple(k.shape[:3])}, got {t.dtype} {tuple(t.shape)}")
    if table.dtype != torch.int32 or table.dim() != 2 or table.numel() == 0:
        raise ValueError(f"table must be int32 of shape (batch, max_pages), not empty, got {table.dtype} {tuple(table.shape)}")
    if lengths.dtype != torch.int32 or tuple(lengths.shape) != (table.shape[0],):
        raise ValueError(f"lengths must be int32 of shape ({table.shape[0]},), got {lengths.dtype} {tuple(lengths.shape)}")
    if table.shape[1] * k.shape[2] > 1 << 28 or table.shape[0] > 0x7fffff or k.shape[1] > 65535 or k.shape[0] > 0x7fffffff:
        raise _lib.FbaError(_lib.FBA_ERR_UNSUPPORTED, f"a sequence may have 2^28 slots at most, a pool 2^31 - 1 pages of 65535 heads, got table {tuple(table.shape)}, cache {tuple(k.shape)}")
    for name, t in (("cache.k", k), ("cache.v", cache.v), ("cache.positions", cache.positions), ("cache.weights", cache.weights)):
        if t is not None and t.data_ptr() % 16:
            raise ValueError(f"{name} must be 16-byte aligned")


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


def cache_append(cache, table, lengths, k, v, counts=None, positions=None, weights=None):
    """Rows of new tokens go to the slots behind `lengths`: k, v (batch, kv_heads, tokens, 128), any strides with dense rows; of sequence b the first counts[b] (int32
    (batch,); None: all).  Where the cache has positions, the tokens' are positions[b], positions[b] + 1, ... (int32 (batch,); None: those of the slots, right
    as long as nothing has been evicted); where it has weights, they begin with `weights` (float32 (batch, kv_heads, tokens); None: zero).

    Returns the new lengths, a tensor of its own: lengths + counts, and -1 where length or count make no sense, there is no room (nothing is written then) or a page is
    outside of the pool (its rows are not written)."""
    given = (cache.k, cache.v, cache.positions, cache.weights, table, lengths) if isinstance(cache, PagedCache) else None
    out = None if given is None else _lib.host().cache_append(*given, k, v, counts, positions, weights)
    if out is not None:
        return out
    _check_cache(cache, table, lengths)
    batch, kv_heads = table.shape[0], cache.k.shape[1]
    for name, t in (("k", k), ("v", v)):
        _require_device(t, name)
        if t.dtype != cache.k.dtype or t.device != cache.k.device:
            raise TypeError(f"{name} must have the cache's type and device ({cache.k.dtype}, {cache.k.device}), got {t.dtype}, {t.device}")
        if t.dim() != 4 or t.shape[0] != batch or t.shape[1] != kv_heads or t.shape[3] != HEAD_DIM or t.shape != k.shape:
            raise ValueError(f"k and v must have shape ({batch}, {kv_heads}, tokens, {HEAD_DIM}), got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.shape[2] > 1 << 28:
        raise _lib.FbaError(_lib.FBA_ERR_UNSUPPORTED, f"a call may append 2^28 tokens at most, got {k.shape[2]}")
    _check_ints(counts, "counts", table)
    _check_ints(positions, "positions", table)
    if positions is not None and cache.positions is None:
        raise ValueError("positions are given, but the cache has none")
    if weights is not None:
        if cache.weights is None:
            raise ValueError("weights are given, but the cache has none")
        if weights.dtype != torch.float32 or weights.shape != k.shape[:3] or weights.device != k.device:
            raise ValueError(f"weights must be float32 of shape {tuple(k.shape[:3])} on {k.device}, got {weights.dtype} {tuple(weights.shape)} on {weights.device}")
    _no_gradients(**{"cache.k": cache.k, "cache.v": cache.v, "cache.weights": cache.weights, "k": k, "v": v, "weights": weights})
    if k.shape[2] == 0:
        right = (lengths >= 0) & (lengths <= table.shape[1] * cache.k.shape[2])
        return torch.where(right if counts is None else right & (counts == 0), lengths, -1)
    dense = lambda t: None if t is None else t.contiguous()
    return _answered(_lib.host().cache_append(*given, _rows_dense(k), _rows_dense(v), dense(counts), dense(positions), dense(weights)))


def cache_attn_func(q, cache, table, lengths, window=None, sinks=0, accumulate=False):
    """Attention of one new token per sequence, the last of its `lengths` slots: softmax(q k^T / sqrt(128)) v over the filled slots or, with `window`, over the last
    `window` of them and the first `sinks`.  (Slots are in the order of tokens as long as nothing has been evicted.)

    q: (batch, heads, 1, 128) of the cache's type, heads a multiple of kv_heads.  accumulate=True adds to cache.weights what softmax gave every slot, summed over the query
    heads of a kv head; not with a window, and with a workspace of 4 * batch * heads bytes for every slot that the table has room for, filled or not.  Returns o, shaped like q: zeros for a sequence without slots, NaN for one whose length or pages make no sense."""
    given = (cache.k, cache.v, cache.weights, table, lengths) if isinstance(cache, PagedCache) else None
    out = None if given is None else _lib.host().cache_attention(q, *given, window, sinks, bool(accumulate))
    if out is not None:
        return out
    _check_cache(cache, table, lengths)
    _require_device(q, "q")
    if q.dtype != cache.k.dtype or q.device != cache.k.device:
        raise TypeError(f"q must have the cache's type and device ({cache.k.dtype}, {cache.k.device}), got {q.dtype}, {q.device}")
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
    return _answered(_lib.host().cache_attention(_rows_dense(q), *given, None if window == _NO_WINDOW else window, sinks, bool(accumulate)))


def cache_evict(cache, table, lengths, budget, recent=0, sinks=0):
    """Brings every sequence of more than `budget` slots down to that, every kv head for itself: tokens at positions below `sinks` and the `recent` last ones stay, then those
    with the largest weights (of equal ones the lower slot; NaN is the lowest).  Slots that are freed below the budget take the kept ones from behind it, in order: rows,
    positions and weights; slots are in no order of tokens then.  batch * kv_heads may be 65535 at most.

    Returns the new lengths, a tensor of its own: min(lengths, budget), and -1, with nothing moved, where a length or page makes no sense."""
    given = (cache.k, cache.v, cache.positions, cache.weights, table, lengths) if isinstance(cache, PagedCache) else None
    out = None if given is None else _lib.host().cache_evict(*given, budget, recent, sinks)
    if out is not None:
        return out
    _check_cache(cache, table, lengths)
    if cache.positions is None or cache.weights is None:
        raise ValueError("eviction needs a cache with positions and weights")
    budget, recent, sinks = _whole(budget, "budget", 1), _whole(recent, "recent", 0), _whole(sinks, "sinks", 0)
    if recent + sinks > budget:
        raise ValueError(f"recent ({recent}) and sinks ({sinks}) must fit the budget ({budget}) together")
    _no_gradients(**{"cache.k": cache.k, "cache.v": cache.v, "cache.weights": cache.weights})
    return _answered(_lib.host().cache_evict(*given, budget, recent, sinks))
