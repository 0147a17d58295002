"""Attention under a sliding window with sinks, at the granularity of tokens: what a block mask (`masks.swa_block_mask`, the sliding tiles and sink blocks of
`video`) cannot say, a border inside a block, and causality.  The kernels are csrc/fba_window_fwd.hip, fba_window_dq.hip, fba_window_dkdv.hip and, for small
calls, fba_window_few.hip; what they compute is stated in include/fba.h."""
import numbers

import torch

from . import _lib
from .interface import HEAD_DIM, _require_device, _typed_like

_NO_WINDOW = 2**31 - 1
_TYPES = (torch.bfloat16, torch.float16)


def _whole(value, name, least):
    if isinstance(value, bool) or not isinstance(value, numbers.Integral):
        raise TypeError(f"{name} must be an integer, got {type(value).__name__}")
    if value < least:
        raise ValueError(f"{name} ({value}) must be at least {least}")
    return min(int(value), _NO_WINDOW)


def _check_window_args(q, k, v, window, sinks, lengths):
    """-> (window, sinks), or an error."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        _require_device(t, name)
        if t.dtype not in _TYPES:
            raise TypeError(f"{name} must be bfloat16 or float16, got {t.dtype}")
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{name} must have q's type and device ({q.dtype}, {q.device}), got {t.dtype}, {t.device}")
        if t.dim() != 4:
            raise ValueError(f"{name} must have shape (batch, heads, seq, head_dim)")
        if t.shape[3] != HEAD_DIM:
            raise ValueError("head_dim must be 128")
    if k.shape[0] != q.shape[0] or v.shape[0] != q.shape[0]:
        raise ValueError("q, k, v batch dimensions must match")
    if v.shape != k.shape:
        raise ValueError("k and v must have the same shape")
    if k.shape[1] == 0 or q.shape[1] % k.shape[1] != 0:
        raise ValueError("q heads must be a multiple of kv heads")
    window = _NO_WINDOW if window is None else _whole(window, "window", 1)
    sinks = _whole(sinks, "sinks", 0)
    if lengths is not None:
        _require_device(lengths, "lengths")
        if lengths.dtype != torch.int32 or lengths.dim() != 1 or lengths.shape[0] != q.shape[0] or lengths.device != q.device:
            raise ValueError(f"lengths must be an int32 tensor of shape ({q.shape[0]},) on {q.device}, got {tuple(lengths.shape)} {lengths.dtype} on {lengths.device}")
        if q.shape[2] != k.shape[2]:
            raise ValueError(f"lengths need q and k of one length, got {q.shape[2]} and {k.shape[2]}")
    return window, sinks


def _rows_dense(t):
    """`t` as the kernels read it: rows dense, everything else at multiples of 16 bytes."""
    strides = [s for s, n in zip(t.stride()[:3], t.shape[:3]) if n > 1]
    fits = t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(s % 8 == 0 and s >= 0 for s in strides) and (t.shape[2] <= 1 or t.stride(2) <= 1 << 24)
    return t if fits else t.clone(memory_format=torch.contiguous_format)


class WindowAttnFunc(torch.autograd.Function):
    """The operator as a Python autograd function: for arguments that need preparation or are refused, calls that are traced and tensor subclasses."""

    @staticmethod
    def forward(ctx, q, k, v, window, sinks, causal, lengths):
        window, sinks = _check_window_args(q, k, v, window, sinks, lengths)
        causal, lengths = bool(causal), None if lengths is None else lengths.contiguous()
        q, k, v = (_rows_dense(t) for t in (q, k, v))
        o, lse, low = _lib.host().window_forward(q, k, v, window, sinks, causal, lengths)
        o = _typed_like(o, q)
        ctx.save_for_backward(q, k, v, o, low, lse)
        # the caller may write to their lengths before backward comes
        ctx.args = (window, sinks, causal, None if lengths is None else lengths.clone())
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, low, lse = ctx.saved_tensors  # (the native side sees to it that this is not differentiated again)
        grads = _lib.host().window_backward(q, k, v, _rows_dense(o), low, lse, do, *ctx.args)
        return (*(_typed_like(g, t) for g, t in zip(grads, (q, k, v))), None, None, None, None)


def window_attn_func(q, k, v, window, sinks=0, causal=True, lengths=None):
    """Attention of every token to the tokens in its window and to the first `sinks` tokens: softmax(q k^T / sqrt(128)) v over the keys j that a row at
    position p sees,

        causal:       j <= p and (p - j < window or j < sinks)
        causal=False: |p - j| < window or j < sinks

    q: (batch, heads, q_seq_len, 128), k, v: (batch, kv_heads, kv_seq_len, 128), bf16 or fp16, heads a multiple of kv_heads.  Any strides: tensors with dense
    rows (a projection's (batch, seq, heads, 128), transposed) are read as they are.  The queries are the last q_seq_len positions of the keys: row i stands at
    i + kv_seq_len - q_seq_len.  `window` None: no limit.  `lengths`, int32 (batch,) on the GPU: sequence b has lengths[b] tokens, the rows behind them are
    padding (not read, zeros in o and in the gradients); q and k then have one length.  A row that sees no key is zeros.

    Scores of keys that a row does not see may be anything; v has to be finite there, and for gradients q, k and the gradient of o too (a weight of zero times infinity is no
    number), padding excepted.  How far such a value reaches, up to 32 rows and 128 keys beside those that see it, is stated in include/fba.h.

    Returns o, shaped like q.  Differentiable in q, k and v, once (differentiating a gradient raises).  Gradients in fp16 need the usual scaling of the
    loss: P and dS, before its factor 1 / sqrt(128), are rounded to the inputs' type, where fp16 ends at 65504 and has fewer digits below 2^-14, for rows whose weight is spread over more
    than some 16000 keys therefore.  A step may be captured into a graph; no earlier
    graph of leaves that the captured backward pass reaches, through views and projections too, may be alive then if it was made on the default stream (backward raises)."""
    o = _lib.host().window_attention(q, k, v, window, sinks, bool(causal), lengths)
    if o is not None:
        return o
    return WindowAttnFunc.apply(q, k, v, window, sinks, causal, lengths)
