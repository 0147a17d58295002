"""Rotary positions against the formula in 64 bits: types, layouts, axes, far coordinates, gradients, captured steps, and beside the operators that they are for.

Tolerance.  With f = 2^-24: a sine or cosine is off by 2^-29 (the series' next term), f for its argument's rounding and some 3 f of its own, 2^-21 with all of it; the two products and
their sum add 2 f of |a| + |b|; the result is rounded once, u = eps / 2 of it, and where fp16 is subnormal by 2^-25:
  |out - exact| <= 2^-20 (|a| + |b|) + u |exact| + 2^-25 (fp16)
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def exact(x, turn, where, inverse=False):
    """(the rotation of x in 64 bits, |a| + |b|), from the whole turns that coordinates make, which integers of 64 bits lose: x (B, H, S, 128), where (B, S, axes) -> float64 on the CPU"""
    x, where = x.detach().double().cpu(), where.cpu().long()
    n = turn.turns.shape[0]
    phase = where[..., turn.axes.cpu().long().clamp_max(turn.n_axes - 1)] * turn.turns.cpu()  # modulo 2^64, a signed fraction of a turn
    angle = (phase.double() * (2 * math.pi / 2**64))[:, None]
    cos, sin = torch.cos(angle), torch.sin(angle) * (-1 if inverse else 1)
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if turn.interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., first], x[..., second]
    out, size = x.clone(), torch.zeros_like(x)
    out[..., first], out[..., second] = a * cos - b * sin, a * sin + b * cos
    size[..., first] = size[..., second] = a.abs() + b.abs()
    return out, size


def check(got, x, turn, where, inverse=False):
    assert got.shape == x.shape and got.dtype == x.dtype and got.device == x.device
    want, size = exact(x, turn, where, inverse)
    off = 2.0**-20 * size + torch.finfo(x.dtype).eps / 2 * want.abs() + (2.0**-25 if x.dtype == torch.float16 else 0.0)
    over = (got.detach().double().cpu() - want).abs() - off
    assert bool((over <= 0).all()), f"{over.max().item():.3e} beyond the bound"
    rest = 2 * turn.turns.shape[0]
    assert torch.equal(got[..., rest:], x[..., rest:])


def random(shape, dtype, gpu, seed=0):
    return torch.randn(shape, generator=torch.Generator(device="cpu").manual_seed(seed)).to(dtype).to(gpu)


def places(kind, B, S, axes, gpu, seed=0):
    """(coordinates as they are given, (B, S, axes) of them)"""
    g = torch.Generator(device="cpu").manual_seed(seed)
    if kind == "none":
        return None, torch.arange(S, dtype=torch.int32)[None, :, None].expand(B, S, axes)
    shape = (S, axes) if kind == "shared" else (B, S, axes)
    where = torch.randint(0, 1000, shape, generator=g, dtype=torch.int32)
    if kind == "far":  # all of 32 bits
        where = torch.randint(-2**31, 2**31, shape, generator=g, dtype=torch.int64).to(torch.int32)
        where.view(-1)[:4] = torch.tensor([-2**31, 2**31 - 1, -1, 0], dtype=torch.int32)[: where.numel()]
    return where.to(gpu), where.expand(B, S, axes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dims,kind,B,H,Hk,S", [
    ((128,), "none", 1, 1, 1, 1), ((128,), "shared", 2, 4, 2, 15), ((16, 56, 56), "each", 2, 3, 1, 33), ((16, 56, 56), "far", 1, 24, 6, 130), ((64,), "none", 3, 5, 5, 17),
    ((96,), "far", 1, 1, 7, 64), ((16,), "shared", 2, 2, 2, 7), ((44, 42, 42), "each", 1, 8, 2, 500), ((32, 16, 16), "none", 1, 130, 3, 9), ((2,) * 8, "far", 2, 3, 3, 40), ((64, 64), "each", 70, 2, 1, 3),
    ((10, 38), "far", 1, 2, 2, 2100),
])
def test_against_the_formula(gpu, dtype, interleaved, dims, kind, B, H, Hk, S):
    import flex_block_attn_amd as fba

    print(f"rotary {dtype} {dims} {'interleaved' if interleaved else 'halves'} {kind} B{B} H{H}/{Hk} S{S}", flush=True)
    turn = fba.rotary(dims, interleaved=interleaved, theta=300.0, device=gpu)
    q, k = random((B, H, S, 128), dtype, gpu, 1), random((B, Hk, S, 128), dtype, gpu, 2)
    given, where = places(kind, B, S, len(dims), gpu)
    before = q.clone(), k.clone()
    for inverse in (False, True):
        gq, gk = fba.rotary_func(q, k, turn, coordinates=given, inverse=inverse)
        check(gq, q, turn, where, inverse)
        check(gk, k, turn, where, inverse)
    alone, none = fba.rotary_func(q, None, turn, coordinates=given, inverse=True)
    assert none is None and torch.equal(alone, gq) and torch.equal(q, before[0]) and torch.equal(k, before[1])


def test_angles_are_those_of_the_frequencies(gpu):
    """Where a product in 64 bits is good enough: positions up to 2^20 times theta^(-2j / 128), off by 2^20 2^-53."""
    import flex_block_attn_amd as fba

    turn = fba.rotary(device=gpu, interleaved=False)
    where = torch.tensor([0, 1, 2, 1000, 2**20 - 1], dtype=torch.int32, device=gpu)[:, None]
    x = torch.zeros((1, 1, 5, 128), dtype=torch.float16, device=gpu)
    x[..., :64] = 1.0
    got, _ = fba.rotary_func(x, None, turn, coordinates=where)
    angle = where.double() * 10000.0 ** (-2 * torch.arange(64, dtype=torch.float64, device=gpu) / 128)
    want = torch.cat([torch.cos(angle), torch.sin(angle)], -1)
    assert float((got[0, 0].double() - want).abs().max()) <= 2.0**-12 + 2.0**-20


def test_an_axis_that_there_is_not_counts_as_the_last(gpu):
    import flex_block_attn_amd as fba

    turn = fba.rotary((16, 16), device=gpu)
    odd = fba.Rotary(turn.turns, torch.tensor([0] * 8 + [7, -1, 100, 2, 1, 1, -2**31, 2**31 - 1], dtype=torch.int32, device=gpu), 2, True)
    x = random((1, 2, 50, 128), torch.bfloat16, gpu)
    given, _ = places("shared", 1, 50, 2, gpu)
    assert torch.equal(fba.rotary_func(x, None, odd, coordinates=given)[0], fba.rotary_func(x, None, turn, coordinates=given)[0])


@pytest.mark.parametrize("interleaved", [False, True])
def test_layouts(gpu, interleaved):
    """Projections, transposed, keep their layout; rows that are not aligned or repeat, and coordinates that are not dense, are taken too."""
    import flex_block_attn_amd as fba

    turn = fba.rotary((32, 32), interleaved=interleaved, device=gpu)
    given, _ = places("each", 2, 37, 2, gpu)
    dense = random((2, 6, 37, 128), torch.bfloat16, gpu)
    want, _ = fba.rotary_func(dense, None, turn, coordinates=given)
    projected = dense.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros((2, 37, 20, 128), dtype=torch.bfloat16, device=gpu)
    wide[:, :, 5:11] = dense.transpose(1, 2)
    odd = torch.nn.functional.pad(dense, (1, 0))[..., 1:]
    columns = dense.transpose(2, 3).contiguous().transpose(2, 3)
    for x in (projected, wide[:, :, 5:11].transpose(1, 2), odd, columns):
        got, _ = fba.rotary_func(x, None, turn, coordinates=given)
        assert torch.equal(got, want)
    assert fba.rotary_func(projected, None, turn)[0].stride() == projected.stride()
    one = dense[:, :1]
    got, same = fba.rotary_func(one.expand(2, 6, 37, 128), one, turn, coordinates=torch.stack([given, given], 2)[:, :, 0])
    assert torch.equal(got, same.expand(2, 6, 37, 128)) and torch.equal(got[:, :1], want[:, :1])


def test_what_is_no_number_stays_in_its_pair(gpu):
    import flex_block_attn_amd as fba

    for interleaved, other in ((False, 3 + 32), (True, 2)):
        turn = fba.rotary((64,), interleaved=interleaved, device=gpu)
        x = random((1, 1, 5, 128), torch.bfloat16, gpu)
        want, _ = fba.rotary_func(x, None, turn)
        bad = x.clone()
        bad[0, 0, 2, 3] = math.nan
        bad[0, 0, 3, 100] = math.inf
        got, _ = fba.rotary_func(bad, None, turn)
        assert bool(got[0, 0, 2, [3, other]].isnan().all()) and got[0, 0, 3, 100] == math.inf
        got[0, 0, 2, [3, other]] = want[0, 0, 2, [3, other]]
        got[0, 0, 3, 100] = want[0, 0, 3, 100]
        assert torch.equal(got, want)


def test_rows_far_into_memory(gpu):
    """Offsets that pass 32 bits, in bytes, of a head and of a sequence."""
    import flex_block_attn_amd as fba

    turn = fba.rotary((16, 56, 56), device=gpu)
    S = 700000
    q = torch.empty((2, 13, S, 128), dtype=torch.bfloat16, device=gpu)
    assert q[0].numel() * 2 > 2**31 and q.numel() * 2 > 2**32
    part = random((2, 13, 100, 128), torch.bfloat16, gpu)
    q.zero_()
    q[:, :, -100:] = part
    given, _ = places("far", 2, S, 3, gpu)
    got, _ = fba.rotary_func(q, None, turn, coordinates=given)
    assert torch.equal(got[:, :, -100:], fba.rotary_func(part, None, turn, coordinates=given[:, -100:].contiguous())[0])
    assert int(got[:, :, :-100].count_nonzero()) == 0


def _ways():
    """Both ways into the operator, and what Python prepares first."""
    import flex_block_attn_amd as fba

    odd = lambda t: torch.nn.functional.pad(t, (1, 0))[..., 1:]
    return {"native": lambda q, k, r, c: fba.rotary_func(q, k, r, coordinates=c), "python": lambda q, k, r, c: fba.RotaryFunc.apply(q, k, r.turns, r.axes, r.n_axes, r.interleaved, c, False),
            "prepared": lambda q, k, r, c: fba.rotary_func(odd(q), odd(k), r, coordinates=c)}


@pytest.mark.parametrize("way", ["native", "python", "prepared"])
@pytest.mark.parametrize("dtype,interleaved", [(torch.bfloat16, True), (torch.float16, False)])
def test_gradients(gpu, way, dtype, interleaved):
    """The gradient is the rotation back: by the formula, and as differences, which of a linear map are as exact at any distance."""
    import flex_block_attn_amd as fba

    f = _ways()[way]
    turn = fba.rotary((32, 64), interleaved=interleaved, device=gpu)
    given, where = places("far", 2, 21, 2, gpu)
    q, k = random((2, 4, 21, 128), dtype, gpu, 1).requires_grad_(True), random((2, 2, 21, 128), dtype, gpu, 2).requires_grad_(True)
    dq, dk = random(q.shape, dtype, gpu, 3), random(k.shape, dtype, gpu, 4)
    out = f(q, k, turn, given)
    grads = torch.autograd.grad(out, (q, k), (dq, dk), retain_graph=True)
    for g, d in zip(grads, (dq, dk)):
        check(g, d, turn, where, inverse=True)
    with torch.no_grad():
        step = random(q.shape, dtype, gpu, 5)
        ahead, behind = f(q + step, k, turn, given)[0], f(q - step, k, turn, given)[0]
        moved = (q + step).double() - (q - step).double()
        slope, want = ((ahead.double() - behind.double()) * dq.double()).sum(), (moved * grads[0].double()).sum()
        u = torch.finfo(dtype).eps / 2 + 2.0**-19  # of the largest that enter, each out rounded once; |row| * |row| bounds a row's products
        off = u * ((ahead.double().norm(dim=-1) + behind.double().norm(dim=-1)) * dq.double().norm(dim=-1) + moved.norm(dim=-1) * dq.double().norm(dim=-1)).sum()
        assert float((slope - want).abs()) <= float(off)
    # one output, one input, a gradient that is broadcast
    assert torch.equal(torch.autograd.grad(out[1], k, dk, retain_graph=True)[0], grads[1])
    only, = torch.autograd.grad(out[0], q, dq, retain_graph=True)
    assert torch.equal(only, grads[0])
    spread, = torch.autograd.grad(out[0].sum(), q, retain_graph=True)
    check(spread, torch.ones_like(q), turn, where, inverse=True)
    with torch.no_grad():
        plain = f(q, k, turn, given)
    assert torch.equal(plain[0], out[0]) and not plain[0].requires_grad
    half = f(q.detach(), k, turn, given)
    assert torch.equal(torch.autograd.grad(half[1], k, dk)[0], grads[1])


@pytest.mark.parametrize("way", ["native", "python", "prepared"])
def test_gradients_of_gradients(gpu, way):
    """The map is linear: the derivative of <rotated back, w> by what is rotated back is w rotated."""
    import flex_block_attn_amd as fba

    f = _ways()[way]
    turn = fba.rotary(device=gpu)
    given, where = places("each", 1, 9, 1, gpu)
    q, k = (random((1, 2, 9, 128), torch.bfloat16, gpu, i).requires_grad_(True) for i in (1, 2))
    d = random(q.shape, torch.bfloat16, gpu, 3).requires_grad_(True)
    w = random(q.shape, torch.bfloat16, gpu, 4)
    for i in (0, 1):
        g, = torch.autograd.grad(f(q, k, turn, given)[i], (q, k)[i], d, create_graph=True)
        again, = torch.autograd.grad(g, d, w)
        check(again, w, turn, where)


def test_saved_tensors_that_were_written_to_raise(gpu):
    import flex_block_attn_amd as fba

    turn = fba.rotary(device=gpu)
    given, _ = places("shared", 1, 9, 1, gpu)
    q = random((1, 2, 9, 128), torch.bfloat16, gpu).requires_grad_(True)
    out, _ = fba.rotary_func(q, None, turn, coordinates=given)
    given.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_a_captured_step(gpu):
    import flex_block_attn_amd as fba

    turn = fba.rotary((16, 56, 56), device=gpu)
    given, _ = places("each", 2, 300, 3, gpu)
    q, k, dq, dk = (random((2, h, 300, 128), torch.bfloat16, gpu, i).requires_grad_(i < 2) for i, h in enumerate((4, 2, 4, 2)))

    def step():
        out = fba.rotary_func(q, k, turn, coordinates=given)
        return (*(t.detach() for t in out), *torch.autograd.grad(out, (q, k), (dq, dk)))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            q.copy_(random(q.shape, torch.bfloat16, gpu, 10 + i))
            dk.copy_(random(dk.shape, torch.bfloat16, gpu, 20 + i))
        given.add_(i)
        want = step()
        torch.cuda.synchronize()
        for t in got:
            t.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("way", ["native", "python"])
def test_capture_beside_an_earlier_graph_of_the_leaves(gpu, way):
    """Refused, as window attention does, while that graph lives: autograd would make its stream wait for the capture, which ends the process."""
    import flex_block_attn_amd as fba

    f = _ways()[way]
    turn = fba.rotary(device=gpu)
    q, k = (random((1, 2, 40, 128), torch.bfloat16, gpu, i).requires_grad_(True) for i in (1, 2))
    dq = random(q.shape, torch.bfloat16, gpu, 3)
    earlier = f(q, k, turn, None)
    want, = torch.autograd.grad(earlier[0], q, dq, retain_graph=True)
    want = want.clone()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="earlier graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(f(q, k, turn, None)[0], q, dq)
    assert torch.equal(torch.autograd.grad(earlier[0], q, dq)[0], want)
    del earlier
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(f(q, k, turn, None)[0], q, dq)
    for _ in range(2):
        got.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_on_two_streams(gpu):
    import flex_block_attn_amd as fba

    turn = fba.rotary(device=gpu)
    xs = [random((1, 8, 3000, 128), torch.bfloat16, gpu, i) for i in (1, 2)]
    want = [fba.rotary_func(x, None, turn)[0] for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(fba.rotary_func(x, None, turn)[0])
    torch.cuda.synchronize()
    for i, t in enumerate(got):
        assert torch.equal(t, want[i % 2])


def test_a_video_layer(gpu):
    """Turned in raster order and tiled, or tiled and turned where the tiles' tokens stand: the same; and through attention with its gradients."""
    import flex_block_attn_amd as fba

    grid, tile = (6, 16, 8), (6, 8, 8)
    turn = fba.rotary((16, 56, 56), theta=256.0, device=gpu)
    q, k, v, do = (random((1, 2, 6 * 16 * 8, 128), torch.bfloat16, gpu, i).requires_grad_(i < 3) for i in range(4))
    raster, tiled = fba.grid_coordinates(grid, device=gpu), fba.grid_coordinates(grid, tile, device=gpu)
    with torch.no_grad():
        a = fba.tile_tokens(fba.rotary_func(q, None, turn, coordinates=raster)[0], grid, tile)
        b = fba.rotary_func(fba.tile_tokens(q, grid, tile), None, turn, coordinates=tiled)[0]
    assert torch.equal(a, b)
    o = fba.ssta_3d_attention(*fba.rotary_func(q, k, turn, coordinates=raster), v, grid, tile, window=(1, 3, 3), topk=2)
    grads = torch.autograd.grad(o, (q, k, v), do)
    # the attention's own gradients, turned back by hand
    rq, rk = (t.detach().requires_grad_(True) for t in fba.rotary_func(q, k, turn, coordinates=raster))
    by_hand = torch.autograd.grad(fba.ssta_3d_attention(rq, rk, v, grid, tile, window=(1, 3, 3), topk=2), (rq, rk, v), do)
    back = fba.rotary_func(*by_hand[:2], turn, coordinates=raster, inverse=True)
    for x, y in zip(grads, (*back, by_hand[2])):
        assert torch.equal(x, y)


def test_calls_that_are_seldom(gpu):
    """Heads and sequences that share memory, coordinates that Python prepares, nothing to turn, inference mode, checkpoints and saved tensors that were elsewhere meanwhile."""
    import flex_block_attn_amd as fba
    from torch.utils.checkpoint import checkpoint

    turn = fba.rotary((64,), interleaved=False, device=gpu)
    q, k = random((2, 4, 33, 128), torch.bfloat16, gpu, 1), random((2, 1, 33, 128), torch.bfloat16, gpu, 2)
    given, where = places("shared", 2, 33, 1, gpu)
    call = lambda q, k, given=given: fba.rotary_func(q, k, turn, coordinates=given)
    want = call(q, k)
    check(want[0], q, turn, where)
    check(want[1], k, turn, where)
    assert torch.equal(call(q, k.expand(-1, 4, -1, -1))[1], want[1].expand(-1, 4, -1, -1))
    for same in (given.expand(2, 33, 1), given.repeat(1, 2)[:, :1]):
        assert torch.equal(call(q, k, same)[0], want[0])
    assert torch.equal(call(torch.cat([q.flatten()[:1], q.flatten()])[1:].view_as(q), None)[0], want[0])  # rows that are not aligned
    assert [tuple(x.shape) for x in call(q[:, :, :0], k[:, :, :0], given[:0])] == [(2, 4, 0, 128), (2, 1, 0, 128)]
    none, some = call(q[:, :0], k)
    assert none.shape == (2, 0, 33, 128) and torch.equal(some, want[1])
    with torch.inference_mode():
        assert torch.equal(call(q.clone(), k)[0], want[0])
    q, k = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    grads = lambda out: torch.autograd.grad([(o.float() ** 2).sum() for o in out], (q, k))
    first = grads(call(q, k))
    again = grads(checkpoint(call, q, k, use_reentrant=False))
    with torch.autograd.graph.save_on_cpu():
        out = call(q, k)
    for x in (again, grads(out)):
        assert all(torch.equal(a, b) for a, b in zip(x, first))
