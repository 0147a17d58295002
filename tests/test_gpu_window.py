"""window_attn_func, forward and gradients, against the formulas in 64 bits, at the sizes and masks where it can go wrong.

Tolerances.  u = eps / 2 of the type: what one rounding is off by.  e: what P is off by, relatively, from fp32 sums: 128 products added in fp32, 130 * 2^-24 of
the sum of their sizes at most, and a few 2^-24 for exp2 and the denominator.
  o   P is rounded once (and its sum with it, u each) and o once:            (2u + 2e) P|v| + u|o|
  dv  P and dv are rounded:                                                  (2u + 2e) P^T|do| + u|dv|
  ds  rounded once; delta comes from the rounded o, dP from fp32 sums:       (2u + 2e) |ds| + P (|do| E_o + 260 * 2^-24 |do||v|)
  dq, dk  the sum of that and a rounding.
P of backward is exp2(S - lse).  With lse of the rounded P's sum, as forward leaves it, it is off by u before it is rounded (all errors of a row are u of the sum together at
most); with that of the sum before, not: the bound covers both.
What is rounded has its own error E by then: a rounding of x + E is off by u (|x| + E) at most, not by u |x|.  Likewise two factors
of 1 + u, and (1 + u) / (1 - u), are off from 1 by 2u + 4u^2 at most.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(128)


def visible(Sq, Skv, window, sinks, causal, length=None, device="cpu"):
    """(Sq, Skv) bool, by the definition."""
    p = torch.arange(Sq, device=device)[:, None] + Skv - Sq
    j = torch.arange(Skv, device=device)[None]
    w = math.inf if window is None else window
    seen = (j <= p) & ((p - j < w) | (j < sinks)) if causal else ((p - j).abs() < w) | (j < sinks)
    if length is not None:
        seen = seen & (j < length) & (p < length)
    return seen


def reference(q, k, v, do, window, sinks, causal, lengths):
    """o, dq, dk, dv in 64 bits, and the bounds of what rounding to the inputs' type may do to each."""
    B, H, Sq, _ = q.shape
    Hk, Skv = k.shape[1:3]
    G = H // Hk
    u, f = torch.finfo(q.dtype).eps / 2, 2.0**-24
    out = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, q, k, v)]
    off = [torch.zeros_like(t) for t in out]
    rows = torch.arange(Sq, device=q.device)
    for b in range(B):
        end = None if lengths is None else min(max(int(lengths[b]), 0), Skv)
        n = Skv if end is None else end
        r = Sq if end is None else end
        seen = visible(Sq, Skv, window, sinks, causal, end, q.device)[:r, :n]
        for h in range(H):
            qd, dod = q[b, h, :r].double(), do[b, h, :r].double()
            kd, vd = k[b, h // G, :n].double(), v[b, h // G, :n].double()
            s = torch.where(seen, qd @ kd.T * SCALE, torch.full(seen.shape, -math.inf, dtype=torch.float64, device=q.device))
            p = torch.softmax(s, -1).nan_to_num(0.0) if n else s
            e = 130 * f * (torch.where(seen, qd.abs() @ kd.abs().T, torch.zeros_like(s)).max().item() if s.numel() else 0.0) * SCALE + 16 * f
            o = p @ vd
            eo = (2 * u + 4 * u * u + 2 * e) * (p @ vd.abs())
            eo = eo + u * (o.abs() + eo)
            delta = (o * dod).sum(-1, keepdim=True)
            ds = p * (dod @ vd.T - delta)
            eds = (2 * u + 4 * u * u + 2 * e) * ds.abs() + p * ((eo * dod.abs()).sum(-1, keepdim=True) + 260 * f * (dod.abs() @ vd.abs().T))
            out[0][b, h, :r], off[0][b, h, :r] = o, eo
            out[1][b, h, :r], off[1][b, h, :r] = ds @ kd * SCALE, eds @ kd.abs() * SCALE
            out[2][b, h // G, :n] += ds.T @ qd * SCALE
            off[2][b, h // G, :n] += eds.T @ qd.abs() * SCALE
            out[3][b, h // G, :n] += p.T @ dod
            off[3][b, h // G, :n] += (2 * u + 4 * u * u + 2 * e) * (p.T @ dod.abs())
    for x, y in list(zip(out, off))[1:]:
        y += u * (x.abs() + y)
    return out, [y + torch.finfo(q.dtype).smallest_normal for y in off]  # (below that fp16 has fixed steps)


def inputs(gpu, B, H, Hk, Sq, Skv, dtype, seed, size=2.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    new = lambda h, n, f=1.0: (torch.randn((B, h, n, 128), generator=g) * f).to(dtype).to(gpu)
    return new(H, Sq, size), new(Hk, Skv), new(Hk, Skv), new(H, Sq)


def check(gpu, q, k, v, do, window, sinks, causal, lengths=None):
    import flex_block_attn_amd as fba

    print(f"window case q{tuple(q.shape)} {q.stride()} k{tuple(k.shape)} window {window} sinks {sinks} causal {causal} lengths {None if lengths is None else lengths.tolist()} {q.dtype}", flush=True)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = fba.window_attn_func(*leaves, window, sinks=sinks, causal=causal, lengths=lengths)
    got = (o.detach(), *torch.autograd.grad(o, leaves, do))
    want, off = reference(q, k, v, do, window, sinks, causal, lengths)
    for name, x, y, z, like in zip(("o", "dq", "dk", "dv"), got, want, off, (q, q, k, v)):
        assert x.dtype == like.dtype and x.shape == like.shape
        assert bool(torch.isfinite(x).all()), name
        over = (x.double() - y).abs() - z
        assert bool((over <= 0).all()), f"{name}: {over.max().item():.3e} beyond the bound, at {(over > 0).sum().item()} of {over.numel()}"
    with torch.no_grad():
        assert torch.equal(fba.window_attn_func(q, k, v, window, sinks=sinks, causal=causal, lengths=lengths), got[0])
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("S,window,sinks", [
    (1, 1, 0), (1, 5, 3), (2, 1, 0), (31, 7, 2), (32, 32, 0), (33, 1, 1), (127, 40, 4), (128, 128, 0), (129, 64, 33), (257, 31, 128), (300, 100, 130), (300, 1, 300),
    (513, 512, 0), (640, 33, 4), (640, None, 0), (777, 200, 97), (1100, 129, 31),
])
def test_lengths_windows_and_sinks(gpu, dtype, causal, S, window, sinks):
    check(gpu, *inputs(gpu, 1, 2, 1, S, S, dtype, S + sinks), window, sinks, causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B,H,Hk,Sq,Skv,window,sinks", [
    (2, 4, 4, 200, 200, 50, 4), (2, 6, 2, 333, 333, 90, 40), (1, 8, 1, 130, 500, 64, 100), (1, 3, 3, 1, 900, 128, 4), (2, 4, 2, 37, 411, None, 0),
    (1, 2, 2, 300, 120, 40, 4),   # more queries than keys: under causality the first ones see nothing
    (1, 2, 1, 200, 1, 3, 1), (1, 2, 2, 500, 260, 1, 0), (1, 24, 6, 150, 150, 33, 16),
])
def test_batches_groups_and_cross_lengths(gpu, causal, B, H, Hk, Sq, Skv, window, sinks):
    check(gpu, *inputs(gpu, B, H, Hk, Sq, Skv, torch.bfloat16, Sq + Skv), window, sinks, causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window,sinks", [(60, 4), (200, 140), (None, 0)])
def test_padded_batches(gpu, causal, window, sinks):
    """Sequences of several lengths, none and more than there is room for among them; what the padding holds is nobody's business."""
    S, lengths = 415, torch.tensor([415, 0, 1, 32, 129, 300, 1000, -3], dtype=torch.int32, device=gpu)
    q, k, v, do = inputs(gpu, len(lengths), 4, 2, S, S, torch.float16, 5)
    for b, n in enumerate(lengths.tolist()):
        for t in (q, k, v, do):
            t[b, :, max(0, n):] = math.nan
    got = check(gpu, q, k, v, do, window, sinks, causal, lengths)
    for x in got:
        for b, n in enumerate(lengths.tolist()):
            assert int(x[b, :, max(0, n):].count_nonzero()) == 0


def test_strides(gpu):
    """A projection's layout, heads of a packed tensor, every second row and tensors that repeat a head: as from contiguous copies, bit for bit."""
    import flex_block_attn_amd as fba

    g = torch.Generator(device="cpu").manual_seed(3)
    packed = torch.randn((2, 300, 3, 4, 128), generator=g).to(torch.bfloat16).to(gpu)
    skipped = torch.randn((2, 4, 600, 128), generator=g).to(torch.bfloat16).to(gpu)
    repeated = torch.randn((2, 1, 300, 128), generator=g).to(torch.bfloat16).to(gpu)
    wide = torch.randn((2, 4, 300, 256), generator=g).to(torch.bfloat16).to(gpu)
    odd = torch.randn((2 * 4 * 300 * 128 + 1,), generator=g).to(torch.bfloat16).to(gpu)[1:].view(2, 4, 300, 128)
    a, b, c = (packed[:, :, i].transpose(1, 2) for i in range(3))
    cases = [(a, b, c), (skipped[:, :, ::2], a, b), (a, repeated.expand(2, 4, 300, 128), c), (wide[..., :128], wide[..., 128:], a), (wide[..., ::2], odd, a)]
    for q, k, v in cases:
        do = torch.randn((2, 300, 4, 128), generator=g).to(torch.bfloat16).to(gpu).transpose(1, 2)
        results = []
        for prepare in (lambda t: t, lambda t: t.contiguous()):
            leaves = [prepare(t).detach().requires_grad_(True) for t in (q, k, v)]
            o = fba.window_attn_func(*leaves, 70, sinks=9)
            results.append((o.detach(), *torch.autograd.grad(o, leaves, prepare(do))))
        for x, y in zip(*results):
            assert torch.equal(x, y)
    # a gradient that repeats one value
    leaf = a.detach().requires_grad_(True)
    x, = torch.autograd.grad(fba.window_attn_func(leaf, b, c, 70, sinks=9).sum(), leaf)
    leaf = a.detach().requires_grad_(True)
    y, = torch.autograd.grad(fba.window_attn_func(leaf, b, c, 70, sinks=9), leaf, torch.ones_like(a).contiguous())
    assert torch.equal(x, y)


@pytest.mark.parametrize("causal", [True, False])
def test_gradients_against_differences(gpu, causal):
    """Along a direction: (f(x + h d) - f(x - h d)) / 2h of f = <o, w> in 64 bits, which is off by h^2 / 6 of the third derivative (1e-6 here), against <grad, d>.  A
    gradient's rounding, and that of P, dS and o, add up over n values as their bounds do, at most."""
    q, k, v, do = inputs(gpu, 1, 2, 1, 150, 150, torch.float16, 8, size=1.0)
    got = check(gpu, q, k, v, do, 40, 5, causal)
    _, off = reference(q, k, v, do, 40, 5, causal, None)
    g = torch.Generator(device="cpu").manual_seed(9)
    seen = visible(150, 150, 40, 5, causal, device=gpu)

    def f(q, k, v):
        s = (q @ k.transpose(-1, -2) * SCALE).masked_fill(~seen, -math.inf)
        return (torch.softmax(s, -1) @ v * do.double()).sum()

    x = [t.double() for t in (q, k, v)]
    for i in range(3):
        d = torch.randn(x[i].shape, generator=g, dtype=torch.float64).to(gpu)
        h = 1e-4
        plus, minus = ([t + s * h * d if j == i else t for j, t in enumerate(x)] for s in (1, -1))
        difference = (f(*plus) - f(*minus)) / (2 * h)
        along = (got[1 + i].double() * d).sum()
        assert abs(difference - along) <= (off[1 + i] * d.abs()).sum() + 1e-5 * (1 + abs(difference))


@pytest.mark.parametrize("H", [1, 80])  # tiles of 32 rows, of 128
def test_masked_places(gpu, H):
    """Keys that a row does not see may hold the type's lowest value, infinities and no numbers in k; in v where no row of their neighbourhood sees them."""
    import flex_block_attn_amd as fba

    S, window, sinks = 512, 64, 4
    q, k, v, _ = inputs(gpu, 1, H, H, S, S, torch.bfloat16, 4)
    # rows 256.. see the sinks and keys from 193 on: what stands between is seen by rows below 160 + 64 only
    want = fba.window_attn_func(q, k, v, window, sinks=sinks)[:, :, 256:]
    for value in (torch.finfo(torch.bfloat16).min, math.inf, -math.inf, math.nan):
        kk, vv = k.clone(), v.clone()
        kk[:, :, 4:160] = value
        vv[:, :, 32:160] = value
        assert torch.equal(fba.window_attn_func(q, kk, vv, window, sinks=sinks)[:, :, 256:], want)
        kk = k.clone()
        kk[:, :, 300:] = value  # in the future of rows below 300
        assert torch.equal(fba.window_attn_func(q, kk, v, window, sinks=sinks)[:, :, 256:300], want[:, :, :44])


def test_nothing_there(gpu):
    import flex_block_attn_amd as fba

    for B, H, Hk, Sq, Skv in ((0, 2, 1, 5, 5), (2, 2, 1, 0, 0), (2, 2, 1, 0, 7), (2, 2, 1, 7, 0), (1, 0, 1, 4, 4)):
        q = torch.randn((B, H, Sq, 128), device=gpu).bfloat16().requires_grad_(True)
        k, v = (torch.randn((B, Hk, Skv, 128), device=gpu).bfloat16().requires_grad_(True) for _ in range(2))
        o = fba.window_attn_func(q, k, v, 4, sinks=1)
        assert o.shape == q.shape and int(o.count_nonzero()) == 0
        for x, t in zip(torch.autograd.grad(o, (q, k, v), torch.ones_like(o)), (q, k, v)):
            assert x.shape == t.shape and int(x.count_nonzero()) == 0


def test_another_stream_and_repeated_calls(gpu):
    """Bit for bit the same, call after call, on a stream of its own, beside another call on the default one."""
    import flex_block_attn_amd as fba

    q, k, v, do = inputs(gpu, 2, 6, 2, 700, 700, torch.bfloat16, 2)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def step():
        o = fba.window_attn_func(*leaves, 130, sinks=20)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            there = step()
        here = step()
        torch.cuda.synchronize()
        for x, y, z in zip(want, there, here):
            assert torch.equal(x, y) and torch.equal(x, z)


def test_step_replays_from_a_captured_graph(gpu):
    """Forward and backward recorded together, lengths and all; replays on new inputs and lengths, with eager steps between."""
    import flex_block_attn_amd as fba

    g = torch.Generator(device="cpu").manual_seed(7)
    new = lambda h: torch.randn((2, h, 500, 128), generator=g).to(torch.bfloat16).to(gpu)
    q, k, v = new(4).requires_grad_(True), new(2).requires_grad_(True), new(2).requires_grad_(True)
    do, lengths = new(4), torch.tensor([500, 333], dtype=torch.int32, device=gpu)

    def step():
        o = fba.window_attn_func(q, k, v, 100, sinks=40, lengths=lengths)
        return (o.detach(), *torch.autograd.grad(o, (q, k, v), do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in ([500, 333], [40, 500], [0, 129]):
        with torch.no_grad():
            for t in (q, k, v, do):
                t.copy_(new(t.shape[1]))
            lengths.copy_(torch.tensor(n, dtype=torch.int32))
        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        for x in out:
            x.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y)


def test_shared_heads_and_one_tensor_for_all(gpu):
    """One tensor as q, k and v: its gradient is the sum of the three."""
    import flex_block_attn_amd as fba

    x = torch.randn((1, 2, 260, 128), device=gpu).bfloat16().requires_grad_(True)
    do = torch.randn_like(x)
    together, = torch.autograd.grad(fba.window_attn_func(x, x, x, 50, sinks=3), x, do)
    leaves = [x.detach().clone().requires_grad_(True) for _ in range(3)]
    parts = torch.autograd.grad(fba.window_attn_func(*leaves, 50, sinks=3), leaves, do)
    # autograd adds the three in bf16, in some order: two roundings of sums that are no larger than the sum of the sizes
    off = 2 * 2.0**-8 * sum(t.double().abs() for t in parts)
    assert bool(((together.double() - sum(t.double() for t in parts)).abs() <= off).all())


def test_writes_nothing_beside_its_outputs(gpu):
    """Through the C ABI, into outputs that are parts of larger tensors: what is around them stays."""
    import ctypes

    from flex_block_attn_amd import _lib
    from flex_block_attn_amd.interface import _stream

    class Strided(ctypes.Structure):
        _fields_ = [("ptr", ctypes.c_void_p), ("batch", ctypes.c_int64), ("head", ctypes.c_int64), ("row", ctypes.c_int64)]

    B, H, Hk, S = 2, 4, 2, 203
    q, k, v, do = inputs(gpu, B, H, Hk, S, S, torch.bfloat16, 6)
    around = [torch.full((B + 2, h, S + 6, 136), 7.0, dtype=torch.bfloat16, device=gpu) for h in (H, H, Hk, Hk)]
    inner = [t[1:-1, :, 3:-3, :128] for t in around]
    stats = torch.full((3 * B * H * S + 64,), 7.0, device=gpu)
    of = lambda t: ctypes.byref(Strided(t.data_ptr(), *t.stride()[:3]))
    sizes = (B, H, Hk, S, S, 128, 40, 5, 1, 0)
    _lib.call("fba_window_fwd", of(q), of(k), of(v), of(inner[0]), None, ctypes.c_void_p(stats.data_ptr()), None, *sizes, _stream())
    n = _lib.load().fba_window_workspace_bytes(0, B, H, Hk, S, S, 40, 5, 1)
    ws = torch.full((n + 64,), 7, dtype=torch.uint8, device=gpu)
    _lib.call("fba_window_bwd", of(q), of(k), of(v), of(inner[0]), None, of(do), ctypes.c_void_p(stats.data_ptr()), None, of(inner[1]), of(inner[2]), of(inner[3]),
              ctypes.c_void_p(ws.data_ptr()), n, *sizes, _stream())
    want, off = reference(q, k, v, do, 40, 5, True, None)
    for t, x, y, z in zip(around, inner, want, off):
        assert bool(((x.double() - y).abs() <= z).all())
        x.fill_(7.0)
        assert bool((t == 7.0).all())
    assert bool((stats[-64:] == 7.0).all()) and bool((ws[n:] == 7).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B,H,Hk,Sq,Skv,window,sinks", [
    (3, 48, 48, 70, 70, 20, 4), (2, 36, 36, 257, 257, 31, 128), (1, 48, 48, 400, 400, 100, 130), (1, 27, 27, 640, 640, 33, 4), (2, 24, 24, 300, 411, None, 0), (2, 48, 48, 300, 120, 40, 4),
    (1, 44, 44, 513, 513, 512, 600), (150, 1, 1, 33, 33, 7, 2), (2, 96, 24, 130, 130, 64, 9), (1, 64, 8, 1100, 1100, 129, 31), (1, 24, 24, 777, 777, 1, 97),
    (4, 100, 100, 70, 70, 20, 4), (2, 66, 33, 257, 257, 31, 128), (1, 98, 49, 400, 400, 100, 130), (1, 78, 6, 640, 640, 33, 4), (2, 66, 66, 300, 411, None, 0), (2, 66, 33, 300, 120, 40, 4),
    (1, 78, 78, 513, 513, 512, 600), (400, 1, 1, 33, 33, 7, 2), (2, 100, 20, 130, 130, 64, 9), (1, 56, 7, 777, 777, 1, 97), (1, 13, 13, 2100, 2100, None, 5),
])
def test_many_rows_and_keys(gpu, dtype, causal, B, H, Hk, Sq, Skv, window, sinks):
    """More than 128 tiles of 128: so are those of dQ, dK and dV, from 256 on those of forward.  (What comes before has tiles of 32.)"""
    check(gpu, *inputs(gpu, B, H, Hk, Sq, Skv, dtype, Sq + H), window, sinks, causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window,sinks", [(60, 4), (200, 140), (None, 0), (1, 31)])
def test_many_rows_and_keys_in_padded_batches(gpu, causal, window, sinks):
    S, lengths = 415, torch.tensor([415, 0, 1, 32, 129, 300, 1000, -3, 257], dtype=torch.int32, device=gpu)
    q, k, v, do = inputs(gpu, len(lengths), 16, 4, S, S, torch.bfloat16, 5)
    for b, n in enumerate(lengths.tolist()):
        for t in (q, k, v, do):
            t[b, :, max(0, n):] = math.nan
    got = check(gpu, q, k, v, do, window, sinks, causal, lengths)
    for x in got:
        for b, n in enumerate(lengths.tolist()):
            assert int(x[b, :, max(0, n):].count_nonzero()) == 0


@pytest.mark.parametrize("B,H,Hk,S,window,sinks,causal", [(1, 4, 1, 2048, 1024, 0, True), (1, 8, 2, 1024, 512, 40, True), (2, 8, 1, 700, 300, 5, False), (1, 1, 1, 1536, 700, 64, False), (1, 8, 2, 2200, 1500, 40, True),
                                                             (1, 8, 2, 2200, 1200, 0, False), (3, 16, 2, 900, 600, 200, True)])
def test_few_keys_with_many_rows_each(gpu, B, H, Hk, S, window, sinks, causal):
    """A tile's rows are cut into several items: tiles of 32 keys, and, where they have more than 4096 rows, of 128."""
    check(gpu, *inputs(gpu, B, H, Hk, S, S, torch.bfloat16, S), window, sinks, causal)


def test_many_rows_in_other_layouts(gpu):
    """As contiguous copies, bit for bit, where tiles have 128 rows."""
    import flex_block_attn_amd as fba

    g = torch.Generator(device="cpu").manual_seed(3)
    packed = torch.randn((2, 300, 3, 70, 128), generator=g).to(torch.bfloat16).to(gpu)
    a, b, c = (packed[:, :, i].transpose(1, 2) for i in range(3))
    do = torch.randn((2, 300, 70, 128), generator=g).to(torch.bfloat16).to(gpu).transpose(1, 2)
    results = []
    for prepare in (lambda t: t, lambda t: t.contiguous()):
        leaves = [prepare(t).detach().requires_grad_(True) for t in (a, b, c)]
        o = fba.window_attn_func(*leaves, 70, sinks=9)
        results.append((o.detach(), *torch.autograd.grad(o, leaves, prepare(do))))
    for x, y in zip(*results):
        assert torch.equal(x, y)


def _both_paths():
    import flex_block_attn_amd as fba

    return fba.window_attn_func, lambda q, k, v, window, sinks: fba.WindowAttnFunc.apply(q, k, v, window, sinks, True, None)


def test_saved_tensors_that_come_back_changed(gpu):
    """From the host and back is the same step; what comes back in another type, shape or place is refused before a kernel reads it."""
    q, k, v, do = inputs(gpu, 1, 4, 2, 100, 100, torch.bfloat16, 3)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    for f in _both_paths():
        want = torch.autograd.grad(f(*leaves, 30, sinks=3), leaves, do)
        with torch.autograd.graph.save_on_cpu():
            o = f(*leaves, 30, sinks=3)
        for x, y in zip(torch.autograd.grad(o, leaves, do), want):
            assert torch.equal(x, y)
        for change, error in ((lambda t: t.cpu(), ValueError), (lambda t: t.double(), TypeError), (lambda t: t[:, :, :50].contiguous(), ValueError), (lambda t: t[..., :64], ValueError)):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
                o = f(*leaves, 30, sinks=3)
            with pytest.raises((error, RuntimeError)):
                torch.autograd.grad(o, leaves, do)
        o = f(*leaves, 30, sinks=3)
        with torch.no_grad():
            k.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(o, leaves, do)


def test_capture_beside_an_earlier_graph_of_the_same_leaves(gpu):
    """Refused by backward, before autograd would make the leaves' stream part of the capture; once the earlier graph is gone the step can be captured."""
    q, k, v, do = inputs(gpu, 1, 4, 2, 100, 100, torch.bfloat16, 3)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    for f in _both_paths():
        earlier = f(*leaves, 30, sinks=3)
        want = (earlier.detach().clone(), *torch.autograd.grad(earlier, leaves, do, retain_graph=True))
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="earlier graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.autograd.grad(f(*leaves, 30, sinks=3), leaves, do)
        for x, y in zip(torch.autograd.grad(earlier, leaves, do), want[1:]):
            assert torch.equal(x, y)
        with torch.cuda.stream(torch.cuda.Stream()):  # outside of a capture another stream is nobody's business
            assert len(torch.autograd.grad(f(*leaves, 30, sinks=3), leaves, do)) == 3
        torch.cuda.synchronize()
        del earlier
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = f(*leaves, 30, sinks=3)
            out = (o.detach(), *torch.autograd.grad(o, leaves, do))
        del o
        for x in out:
            x.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y)


def test_rows_and_batches_far_apart(gpu):
    """Offsets in bytes beyond 32 bits, by the rows' stride (the largest there may be), and by the batches'."""
    import flex_block_attn_amd as fba

    step, S = 1 << 24, 150
    buf = torch.zeros(S * step, dtype=torch.bfloat16, device=gpu)  # 5 GB
    assert 2 * (S - 1) * step > 2**32
    g = torch.Generator(device="cpu").manual_seed(1)
    by_rows = [buf.as_strided((1, 2, S, 128), (0, 512, step, 1), 128 * i) for i in range(4)]
    last = S * step - 2**18
    by_batches = [buf.as_strided((2, 2, S, 128), (last, 128 * S, 128, 1), 2**16 * i) for i in range(4)]
    for views in (by_rows, by_batches):
        new = [torch.randn(v.shape, generator=g).to(torch.bfloat16).to(gpu) for v in views]
        for v, x in zip(views, new):
            v.copy_(x)
        results = []
        for prepare in (lambda t: t, lambda t: t.contiguous()):
            leaves = [prepare(t).detach().requires_grad_(True) for t in views[:3]]
            o = fba.window_attn_func(*leaves, 70, sinks=9)
            results.append((o.detach(), *torch.autograd.grad(o, leaves, prepare(views[3]))))
        for x, y in zip(*results):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,S", [(2, 300), (140, 300)])
def test_large_scores(gpu, dtype, H, S):
    """So large that one key has all the weight: finite, a row of v each, and no gradient to speak of in q and k."""
    import flex_block_attn_amd as fba

    q, k, v, do = inputs(gpu, 1, H, H, S, S, dtype, 3, size=1.0)
    leaves = [t.requires_grad_(True) for t in (q * 1000, k, v)]
    o = fba.window_attn_func(*leaves, 40, sinks=3)
    grads = torch.autograd.grad(o, leaves, do)
    s = (leaves[0].detach().double() @ k.detach().double().transpose(-1, -2) * SCALE).masked_fill(~visible(S, S, 40, 3, True, device=gpu), -math.inf)
    top = s.topk(2, -1)
    clear = top.values[..., 0] - top.values[..., 1] > 40  # the second one's weight is below 2^-57
    assert int(clear.sum()) > clear.numel() // 2
    best = torch.gather(v.detach(), 2, top.indices[..., :1].expand(-1, -1, -1, 128))
    assert torch.equal(o[clear], best[clear])
    for x in grads:
        assert bool(torch.isfinite(x).all())


def test_graphs_that_replay_in_turn_on_two_streams(gpu):
    """Whole steps; each graph has its own workspaces."""
    import flex_block_attn_amd as fba

    sets = [[t.requires_grad_(i < 3) for i, t in enumerate(inputs(gpu, 1, 4, 2, 400, 400, torch.bfloat16, seed))] for seed in (1, 2)]

    def step(q, k, v, do):
        o = fba.window_attn_func(q, k, v, 60, sinks=40)
        return (o.detach(), *torch.autograd.grad(o, (q, k, v), do))

    want = [[x.clone() for x in step(*s)] for s in sets]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(*s))
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(4):
        for out in outs:
            for x in out:
                x.fill_(math.nan)
        for s, graph in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            for x, y in zip(out, w):
                assert torch.equal(x, y)
