"""The paged cache in 4 bits, the rotation on the way into a cache and rows read back, against plain implementations.

What is held is compared exactly: 4 bits of a value are found here by the distances to all fifteen values in 64 bits, and a rotated key is turned in 64 bits on both sides (random values
come within 2^-50 of a border between two codes, where the sides may differ, once in some 2^45 times).  A key that is turned and kept in 16 bits has the bound of test_gpu_rotary.py, and
attention over 4 bits that of test_gpu_cache.py over the values that they stand for, which the type holds.
"""
import math
from dataclasses import replace

import pytest
import torch

from test_gpu_cache import attend_reference, evict_reference, rows
from test_gpu_rotary import check as check_turned
from test_gpu_rotary import exact

pytestmark = pytest.mark.gpu

STEPS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
LIMIT = {torch.bfloat16: 125, torch.float16: 13}


def held(x, dtype):
    """x (..., 128) float64 on the CPU -> (values that 4 bits hold of it, scales (..., 4))"""
    groups = x.reshape(-1, 32)
    values, scales = torch.empty_like(groups), []
    for i, row in enumerate(groups):
        most = float(row.abs().max())
        if not math.isfinite(most):
            values[i] = math.nan
            scales.append(255)
            continue
        e = math.frexp(most)[1] - 3 if most > 0 else -LIMIT[dtype]  # most = m 2^(e + 3), m from 0.5 to 1: e + 2 is the binade
        if most >= 1.75 * 2.0 ** (e + 2):
            e += 1
        e = max(-LIMIT[dtype], min(LIMIT[dtype], e))
        scales.append(e + 127)
        far = (row.abs()[:, None] / 2.0**e - STEPS).abs()
        near = far.amin(1, keepdim=True)
        even = far.masked_fill(torch.arange(8) % 2 == 1, math.inf)
        code = torch.where(even.amin(1) == near[:, 0], even.argmin(1), far.argmin(1))
        values[i] = torch.where(row < 0, -STEPS[code], STEPS[code]) * 2.0**e
    return values.reshape(x.shape), torch.tensor(scales).reshape(*x.shape[:-1], 4)


def decoded(codes, scales):
    """What a pool's bytes stand for, in 64 bits, where they are."""
    nibbles = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    steps = torch.cat([STEPS, -STEPS]).to(codes.device)
    unit = torch.where(scales == 255, torch.full(scales.shape, math.nan, dtype=torch.float64, device=codes.device), torch.exp2(scales.double() - 127))
    return steps[nibbles] * unit.repeat_interleave(32, -1)


def wide(cache):
    """The cache that holds the same values in 16 bits."""
    import flex_block_attn_amd as fba

    return fba.PagedCache(decoded(cache.k, cache.k_scales).to(cache.dtype), decoded(cache.v, cache.v_scales).to(cache.dtype), cache.positions, cache.weights)


def make(gpu, B, Hk, most, page, dtype=torch.bfloat16, seed=0, spare=3, extra=0):
    """(cache with everything, table): pages dealt out of order; what is not filled is no number."""
    import flex_block_attn_amd as fba

    g = torch.Generator(device="cpu").manual_seed(seed)
    per = -(-most // page) + extra
    pages = B * per + spare
    cache = fba.paged_cache(pages, Hk, page, dtype=dtype, device=gpu, evicting=True, bits=4)
    for t in (cache.k, cache.v, cache.k_scales, cache.v_scales):
        t.fill_(255)
    cache.weights.fill_(math.nan)
    cache.positions.fill_(-7)
    table = torch.randperm(pages, generator=g)[: B * per].to(torch.int32).reshape(B, per).to(gpu)
    return cache, table, g


def fill(cache, table, lengths, g):
    """Random codes and scales of sizes around one, weights and positions, in the filled slots of every sequence."""
    page = cache.k.shape[2]
    for b, n in enumerate(lengths):
        for i in range(-(-max(0, n) // page)):
            m, at = min(page, n - i * page), int(table[b, i])
            shape = (cache.k.shape[1], m)
            for codes, scales in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
                codes[at, :, :m] = torch.randint(0, 256, (*shape, 64), generator=g).to(codes)
                scales[at, :, :m] = torch.randint(123, 127, (*shape, 4), generator=g).to(scales)
            cache.weights[at, :, :m] = (torch.rand(shape, generator=g) * 3).to(cache.weights)
            cache.positions[at, :, :m] = torch.arange(i * page, i * page + m, dtype=torch.int32).to(cache.positions)


def ints(x, gpu):
    return torch.tensor(x, dtype=torch.int32, device=gpu)


def every(cache):
    return {name: t for name, t in vars(cache).items() if isinstance(t, torch.Tensor)}


# ---------------------------------------------------------------------------------------------------------------------
# into 4 bits
# ---------------------------------------------------------------------------------------------------------------------
def sample(kind, shape, dtype, g):
    x = torch.randn(shape, generator=g)
    if kind == "ties":  # on the borders between two codes, with a largest value that sets the scale
        borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.0, 0.5, 6.0, 6.9])
        x = borders[torch.randint(0, len(borders), shape, generator=g)] * torch.randint(0, 2, shape, generator=g).sub(0.5).sign()
        x.view(-1, 32)[:, 5] = torch.tensor([4.0, 6.0, 6.5, 6.96875])[torch.randint(0, 4, (x.numel() // 32,), generator=g)]
        x = x * 2.0 ** torch.randint(-8, 8, shape[:-1], generator=g)[..., None]
    elif kind == "scales":  # groups from the smallest normal numbers of the type to the largest, and of zeros
        low, high = (-14, 15) if dtype == torch.float16 else (-126, 127)
        x = (x.double() * 2.0 ** torch.randint(low, high + 1, (*shape[:-1], 4), generator=g).double().repeat_interleave(32, -1))
        top = torch.finfo(dtype).max
        x = x.clamp(-top, top).to(dtype).float()
        x[x.abs() < torch.finfo(dtype).tiny] = 0.0
        x.view(-1, 32)[::7] = 0.0
        x.view(-1, 32)[3::11, 1] = top
    elif kind == "largest":  # around 1.75 of a binade, where the scale changes
        x = x.clamp(-1.5, 1.5)
        x.view(-1, 32)[:, 31] = 1.75 + (torch.randint(-3, 4, (x.numel() // 32,), generator=g) * torch.finfo(dtype).eps)
    elif kind == "numbers that are none":
        x.view(-1, 32)[::3, 7] = math.nan
        x.view(-1, 32)[1::5, 30] = math.inf
        x.view(-1, 32)[2::9, 0] = -math.inf
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["normal", "ties", "scales", "largest", "numbers that are none"])
def test_what_4_bits_hold(gpu, dtype, kind):
    import flex_block_attn_amd as fba

    B, Hk, T = 2, 3, 37
    cache, table, g = make(gpu, B, Hk, 50, 16, dtype)
    k, v = sample(kind, (B, Hk, T, 128), dtype, g), sample(kind, (B, Hk, T, 128), dtype, g)
    n = fba.cache_append(cache, table, ints([5, 0], gpu), k.to(gpu), v.to(gpu))
    assert n.tolist() == [42, 37]
    back = fba.cache_read(cache, table, n, 45)
    for codes, scales, x, got in ((cache.k, cache.k_scales, k, back[0]), (cache.v, cache.v_scales, v, back[1])):
        values, want = held(x.double(), dtype)
        for b, first in ((0, 5), (1, 0)):
            c, s = rows(codes, table, b, first + T)[:, first:], rows(scales, table, b, first + T)[:, first:]
            assert torch.equal(s.cpu().long(), want[b])
            assert torch.equal(decoded(c, s).cpu().nan_to_num(-5.0), values[b].nan_to_num(-5.0))
            assert got.dtype == dtype and torch.equal(got[b, :, first:first + T].double().cpu().nan_to_num(-5.0), values[b].nan_to_num(-5.0))
        assert int(got[1, :, 37:].count_nonzero()) == 0
        # as stated: off by a quarter of the scale or of the value at most, up to 7 times the largest scale
        unit = torch.exp2(want.double() - 127).repeat_interleave(32, -1)
        fits = x.double().abs() <= 7 * 2.0 ** LIMIT[dtype]
        right = (values - x.double()).abs() <= torch.maximum(unit, x.double().abs()) / 4
        assert bool((right | ~fits | (want == 255).repeat_interleave(32, -1)).all())


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dims,interleaved,where,page,before,counts,H", [
    ((128,), False, "slots", 16, [0, 5, 16, 40], [1, 1, 1, 1], 6), ((16, 56, 56), True, "each", 16, [0, 5, 16, 40], [37, 0, 16, 3], 3), ((64,), False, "positions", 64, [63, 64, 65], [200, 129, 1], 0),
    ((16, 32), False, "shared", 256, [10], [400], 9), ((128,), True, "positions", 16, [3] * 70, [1] * 70, 6), ((96,), False, "slots", 32, [0, 7], [70, 70], 40),
])
def test_append_with_the_rotation(gpu, bits, dtype, dims, interleaved, where, page, before, counts, H):
    import flex_block_attn_amd as fba

    B, Hk, T = len(before), 3, max(counts)
    most = max(a + c for a, c in zip(before, counts))
    cache, table, g = make(gpu, B, Hk, most, page, dtype)
    if bits == 16:
        cache = fba.PagedCache(torch.full((*cache.k.shape[:3], 128), math.nan, dtype=dtype, device=gpu), torch.full((*cache.k.shape[:3], 128), math.nan, dtype=dtype, device=gpu), cache.positions, cache.weights)
    print(f"append {bits} bits {dtype} {dims} {where} page {page} before {before[:4]} counts {counts[:4]} heads {H}", flush=True)
    turn = fba.rotary(dims, interleaved=interleaved, device=gpu)
    k, v = (torch.randn((B, T, Hk, 128), generator=g).to(dtype).to(gpu).transpose(1, 2) for _ in range(2))
    q = torch.randn((B, T, H, 128), generator=g).to(dtype).to(gpu).transpose(1, 2) if H else None
    axes = len(dims)
    first = [10**9 + 1000 * b for b in range(B)] if where == "positions" else before
    stand = (torch.tensor(first)[:, None] + torch.arange(T))[..., None].expand(B, T, axes)
    given = None
    if where in ("each", "shared"):
        given = torch.randint(-2**31, 2**31, (B, T, axes) if where == "each" else (T, axes), generator=g).to(torch.int32).to(gpu)
        stand = given.expand(B, T, axes)
    weights = torch.rand((B, Hk, T), generator=g).to(gpu)
    before_all = {name: t.clone() for name, t in every(cache).items()}
    out, turned = fba.cache_append_rotary(cache, table, ints(before, gpu), k, v, turn, q=q, counts=ints(counts, gpu), positions=ints(first, gpu) if where == "positions" else None,
                                          weights=weights, coordinates=given)
    assert out.tolist() == [a + c for a, c in zip(before, counts)]
    if H:
        check_turned(turned, q, turn, stand)
        assert turned.stride() == q.stride()
    else:
        assert turned is None
    want_k, _ = exact(k, turn, stand)
    untouched = {name: torch.ones(t.shape[:3], dtype=torch.bool, device=gpu) for name, t in every(cache).items()}
    for b, (n, c) in enumerate(zip(before, counts)):
        slot = torch.arange(n, n + c, device=gpu)
        pages, at = table[b].long()[slot // page], slot % page
        pick = lambda t: t[pages, :, at].transpose(0, 1)
        if bits == 4:
            for x, codes, scales in ((want_k[b, :, :c], cache.k, cache.k_scales), (v[b, :, :c].double().cpu(), cache.v, cache.v_scales)):
                values, s = held(x, dtype)
                assert torch.equal(pick(scales).cpu().long(), s) and torch.equal(decoded(pick(codes), pick(scales)).cpu(), values)
        else:
            check_turned(pick(cache.k)[None], k[b:b + 1, :, :c], turn, stand[b:b + 1, :c])
            assert torch.equal(pick(cache.v), v[b, :, :c])
        assert torch.equal(pick(cache.positions), (first[b] + torch.arange(c, dtype=torch.int32, device=gpu)).expand(Hk, c))
        assert torch.equal(pick(cache.weights), weights[b, :, :c])
        for m in untouched.values():
            m[pages, :, at] = False
    for name, t in every(cache).items():  # all other slots as they were
        x, y = t[untouched[name]], before_all[name][untouched[name]]
        assert torch.equal(x.nan_to_num(-5.0) if x.is_floating_point() else x, y.nan_to_num(-5.0) if y.is_floating_point() else y), name
    # the same without positions and weights in the cache, and rows that Python prepares
    bare = replace(cache, positions=None, weights=None, k=cache.k.clone(), v=cache.v.clone())
    odd = lambda t: None if t is None else torch.nn.functional.pad(t, (1, 0))[..., 1:]
    again, same = fba.cache_append_rotary(bare, table, ints(before, gpu), odd(k), odd(v), turn, q=odd(q), counts=ints(counts, gpu), positions=ints(first, gpu), coordinates=given)
    assert torch.equal(again, out) and torch.equal(bare.k.view(torch.int8), cache.k.view(torch.int8)) and torch.equal(bare.v.view(torch.int8), cache.v.view(torch.int8)) and (q is None or torch.equal(same, turned))


def held_at_once(x, dtype):
    """`held`, all groups at a time, on x's device.  Exact: a power of two, a difference of two numbers of few bits and a comparison each."""
    groups = x.reshape(-1, 32)
    most = groups.abs().amax(1)
    e = torch.frexp(most)[1].long() - 3
    e = torch.where(most >= 1.75 * torch.exp2((e + 2).double()), e + 1, e)
    e = torch.where(most > 0, e, torch.full_like(e, -LIMIT[dtype])).clamp(-LIMIT[dtype], LIMIT[dtype])
    unit = torch.exp2(e.double())[:, None]
    small = groups.abs() / unit
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=x.device)
    up = torch.tensor([False, True, False, True, False, True, False], device=x.device)  # a tie goes to the even code
    code = ((small[..., None] > borders) | ((small[..., None] == borders) & up)).sum(-1)
    values = torch.where(groups < 0, -1.0, 1.0) * STEPS.to(x.device)[code] * unit
    return values.reshape(x.shape), (e + 127).reshape(*x.shape[:-1], 4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kind", ["many", "quarter turns", "small", "large"])
def test_a_turned_key_is_held_as_64_bits_say(gpu, dtype, interleaved, kind):
    """Where 32 bits would not do: many values, of which some come near to a border between two codes; values on the borders, at rest or turned by whole quarters, which both sides do
    exactly; values around the smallest and the largest normal numbers of the type."""
    import flex_block_attn_amd as fba

    B, Hk, T, page = 2, 3, 2000 if kind == "many" else 150, 64
    cache, table, g = make(gpu, B, Hk, T, page, dtype)
    turn = fba.rotary((32, 64) if kind == "many" else (128,), interleaved=interleaved, device=gpu)
    stand = torch.randint(-5000, 5000, (B, T, turn.n_axes), generator=g, dtype=torch.int32).to(gpu)
    k = torch.randn((B, Hk, T, 128), generator=g)
    if kind == "quarter turns":
        turn.turns.fill_(2**62)
        k = sample("ties", (B, Hk, T, 128), dtype, g)
    elif kind == "small":  # (fp16 holds no more than 2^-15 of its smallest scale's codes)
        k = k * 2.0 ** torch.randint(*((-14, -8) if dtype == torch.float16 else (-120, -96)), (B, Hk, T, 1), generator=g)
        k = torch.where(k.abs() < torch.finfo(dtype).tiny, 0.0, k)
        k[:, :, ::5] = 0.0
    elif kind == "large":
        top = torch.finfo(dtype).max
        k = (k.double() * top).clamp(-top, top)
    k = k.to(dtype).to(gpu)
    print(f"held turned {dtype} {interleaved} {kind}", flush=True)
    n, _ = fba.cache_append_rotary(cache, table, ints([0] * B, gpu), k, k, turn, coordinates=stand)
    assert n.tolist() == [T] * B
    if kind == "quarter turns":
        x = k.double()
        first, second = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, 64), slice(64, 128))
        quarter = (stand % 4)[:, None]  # (B, 1, T, 1)
        a, b = x[..., first], x[..., second]
        want = x.clone()
        pick = lambda *of: torch.where(quarter == 0, of[0], torch.where(quarter == 1, of[1], torch.where(quarter == 2, of[2], of[3])))
        want[..., first], want[..., second] = pick(a, -b, -a, b), pick(b, a, -b, -a)
    else:
        want = exact(k, turn, stand)[0].to(gpu)
    values, scales = held_at_once(want, dtype)
    some = want[:1, :1, :40].cpu()
    assert torch.equal(held(some, dtype)[0], values[:1, :1, :40].cpu()) and torch.equal(held(some, dtype)[1], scales[:1, :1, :40].cpu())
    tiny = torch.finfo(dtype).tiny if dtype == torch.bfloat16 else 0.0
    for b in range(B):
        c, s = rows(cache.k, table, b, T), rows(cache.k_scales, table, b, T)
        assert torch.equal(s.long(), scales[b])
        got = decoded(c, s)
        assert bool(((got == values[b]) | (want[b].abs() < tiny) & (got == 0)).all())


@pytest.mark.parametrize("bits", [4, 16])
def test_append_where_there_is_no_room(gpu, bits):
    """Lengths, counts and pages that make no sense are answered with -1 and a q of no numbers: nothing is written but rows on good pages of a table with a bad one."""
    import flex_block_attn_amd as fba

    cache, table, g = make(gpu, 6, 2, 64, 16)
    if bits == 16:
        cache = fba.PagedCache(torch.zeros((*cache.k.shape[:3], 128), dtype=torch.bfloat16, device=gpu), torch.zeros((*cache.k.shape[:3], 128), dtype=torch.bfloat16, device=gpu), cache.positions, cache.weights)
    table[4, 1] = -3
    before = {name: t.clone() for name, t in every(cache).items()}
    k, v = (torch.randn((6, 2, 20, 128), generator=g).to(torch.bfloat16).to(gpu) for _ in range(2))
    q = torch.randn((6, 3, 20, 128), generator=g).to(torch.bfloat16).to(gpu)
    turn = fba.rotary(device=gpu)
    n, c = ints([45, 65, -1, 10, 10, 44], gpu), ints([20, 1, 1, 21, 20, 20], gpu)
    out, turned = fba.cache_append_rotary(cache, table, n, k, v, turn, q=q, counts=c)
    assert out.tolist() == [-1, -1, -1, -1, -1, 64]
    assert bool(turned[:4].isnan().all()) and bool(turned[4:].isfinite().all())
    for t in range(4):
        for p in table[t].tolist():
            for name, x in every(cache).items():
                x, y = x[p], before[name][p]
                assert torch.equal(x.nan_to_num(-5.0) if x.is_floating_point() else x, y.nan_to_num(-5.0) if y.is_floating_point() else y)
    assert fba.cache_append_rotary(cache, table, out, k, v, turn)[0].tolist()[:5] == [-1] * 5
    if bits == 4:
        assert fba.cache_append(cache, table, out, k, v).tolist()[:5] == [-1] * 5


# ---------------------------------------------------------------------------------------------------------------------
# out of a cache
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,page,slots,first", [([1, 0, 100, 64], 16, 100, 0), ([63, 64, 65], 64, 65, 1), ([300], 256, 1, 299), ([5, 129], 32, 200, 60), ([40], 16, 500, 100)])
def test_read(gpu, bits, dtype, lengths, page, slots, first):
    import flex_block_attn_amd as fba

    cache, table, g = make(gpu, len(lengths), 3, max(lengths), page, dtype, extra=1)
    fill(cache, table, lengths, g)
    values = wide(cache)
    k, v = fba.cache_read(cache if bits == 4 else values, table, ints(lengths, gpu), slots, first=first)
    for got, pool in ((k, values.k), (v, values.v)):
        assert got.shape == (len(lengths), 3, slots, 128) and got.dtype == dtype
        for b, n in enumerate(lengths):
            m = max(0, min(n, first + slots) - first)
            assert torch.equal(got[b, :, :m], rows(pool, table, b, n)[:, first:first + m])
            assert int(got[b, :, m:].count_nonzero()) == 0


@pytest.mark.parametrize("bits", [4, 16])
def test_read_of_wrong_lengths_and_pages(gpu, bits):
    import flex_block_attn_amd as fba

    cache, table, g = make(gpu, 4, 2, 64, 16)
    fill(cache, table, [64] * 4, g)
    cache = cache if bits == 4 else wide(cache)
    good = fba.cache_read(cache, table, ints([64] * 4, gpu), 70)
    table[1, 2], table[3, 3] = cache.k.shape[0], 1 << 30
    k, v = fba.cache_read(cache, table, ints([65, 64, -1, 48], gpu), 70)
    for got, want in ((k, good[0]), (v, good[1])):
        assert bool(got[[0, 2]].isnan().all()) and bool(got[1, :, 32:48].isnan().all())
        assert torch.equal(got[1, :, :32], want[1, :, :32]) and torch.equal(got[1, :, 48:], want[1, :, 48:])
        assert torch.equal(got[3, :, :48], want[3, :, :48]) and int(got[3, :, 48:].count_nonzero()) == 0


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
def check_attend(q, cache, table, lengths, window=None, sinks=0, accumulate=False):
    import flex_block_attn_amd as fba

    print(f"attend q{tuple(q.shape)} cache{tuple(cache.k.shape)} table{tuple(table.shape)} lengths {lengths[:8]} window {window} sinks {sinks} accumulate {accumulate} {q.dtype}", flush=True)
    want, off, added, added_off = attend_reference(q, wide(cache), table, lengths, window, sinks)
    before = cache.weights.clone()
    o = fba.cache_attn_func(q, cache, table, ints(lengths, q.device), window=window, sinks=sinks, accumulate=accumulate)
    assert o.shape == q.shape and o.dtype == q.dtype
    over = (o.double() - want).abs() - off
    assert bool((over <= 0).all()), f"{over.max().item():.3e} beyond the bound"
    if accumulate:
        expected = before.clone()
        for b, m in enumerate(lengths):
            y = rows(before, table, b, m).double() + added[b]
            x = rows(cache.weights, table, b, m).double()
            assert bool(((x - y).abs() <= added_off[b] + 2 * 2.0**-24 * y.abs()).all())
            s = torch.arange(m, device=q.device)
            expected[table[b].long()[s // cache.k.shape[2]], :, s % cache.k.shape[2]] = x.float().transpose(0, 1)
        assert torch.equal(expected.nan_to_num(-5.0), cache.weights.nan_to_num(-5.0))  # all other slots as they were
    else:
        assert torch.equal(before.nan_to_num(-5.0), cache.weights.nan_to_num(-5.0))
    return o


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,H,Hk,page", [
    ([1], 1, 1, 16), ([0, 1, 2], 2, 1, 16), ([15, 16, 17, 31, 32, 33], 8, 2, 16), ([63, 64, 65, 127, 129], 6, 6, 64), ([255, 256, 257, 1000], 12, 4, 32),
    ([5000, 3, 0, 777], 16, 1, 128), ([2049], 17, 1, 16), ([700, 300], 33, 1, 256), ([700, 300], 70, 1, 32), ([640], 130, 2, 64), ([9001, 4000], 24, 6, 64),
    ([5000, 4096, 1], 8, 2, 4096),
])
def test_attend(gpu, dtype, accumulate, lengths, H, Hk, page):
    cache, table, g = make(gpu, len(lengths), Hk, max(lengths + [1]), page, dtype, seed=sum(lengths), extra=1)
    fill(cache, table, lengths, g)
    q = (torch.randn((len(lengths), H, 1, 128), generator=g) * 2).to(dtype).to(gpu)
    check_attend(q, cache, table, lengths, accumulate=accumulate)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 4), (32, 32), (33, 0), (100, 40), (300, 1), (1000, 64), (5000, 0), (20, 3000)])
def test_attend_in_a_window(gpu, window, sinks):
    """Slots between the sinks and the window hold no numbers here: they are not seen."""
    lengths = [0, 1, 31, 64, 100, 333, 1500]
    cache, table, g = make(gpu, len(lengths), 2, max(lengths), 16, seed=window)
    fill(cache, table, lengths, g)
    for b, n in enumerate(lengths):
        for s in range(sinks, max(sinks, n - window)):
            at = int(table[b, s // 16])
            cache.k_scales[at, :, s % 16, s % 4] = 255
            cache.v_scales[at, :, s % 16, s % 3] = 255
    q = (torch.randn((len(lengths), 6, 1, 128), generator=g) * 2).to(torch.bfloat16).to(gpu)
    check_attend(q, cache, table, lengths, window=window, sinks=sinks)


@pytest.mark.parametrize("B", [63, 64, 65, 200])
def test_attend_many_sequences(gpu, B):
    lengths = [(37 * i) % 211 for i in range(B)]
    cache, table, g = make(gpu, B, 2, max(lengths), 16, seed=B)
    fill(cache, table, lengths, g)
    q = torch.randn((B, 4, 1, 128), generator=g).to(torch.bfloat16).to(gpu)
    check_attend(q, cache, table, lengths, accumulate=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attend_all_scales(gpu, dtype):
    """The smallest and the largest scales, in one row: values, not scales, are what is multiplied."""
    cache, table, g = make(gpu, 2, 2, 300, 16, dtype)
    fill(cache, table, [300, 77], g)
    some = cache.v_scales != 255
    low, high = (127 - 13, 127 + 4) if dtype == torch.float16 else (127 - 125, 127 + 100)  # (the largest: P in 16 bits times |v| has to fit)
    scales = torch.randint(low, high + 1, cache.v_scales.shape, generator=g).to(cache.v_scales)
    cache.v_scales.copy_(torch.where(some, scales, cache.v_scales))
    q = torch.randn((2, 4, 1, 128), generator=g).to(dtype).to(gpu)
    check_attend(q, cache, table, [300, 77])
    check_attend(q * 100, cache, table, [300, 77])


def test_a_value_that_is_none_reaches_its_sequence(gpu):
    """A seen key that is no number answers its head with none, and no other; a seen value its columns."""
    import flex_block_attn_amd as fba

    cache, table, g = make(gpu, 3, 2, 100, 16)
    fill(cache, table, [100] * 3, g)
    q = torch.randn((3, 4, 1, 128), generator=g).to(torch.bfloat16).to(gpu)
    n = ints([100] * 3, gpu)
    want = fba.cache_attn_func(q, cache, table, n)
    cache.k_scales[int(table[0, 2]), 1, 3, 2] = 255
    cache.v_scales[int(table[2, 0]), 0, 9, 1] = 255
    o = fba.cache_attn_func(q, cache, table, n)
    assert bool(o[0, 2:].isnan().all()) and bool(o[2, :2, :, 32:64].isnan().all())
    for got, same in ((o[0, :2], want[0, :2]), (o[1], want[1]), (o[2, 2:], want[2, 2:]), (o[2, :2, :, :32], want[2, :2, :, :32]), (o[2, :2, :, 64:], want[2, :2, :, 64:])):
        assert torch.equal(got, same)


@pytest.mark.parametrize("accumulate", [False, True])
def test_wrong_lengths_and_pages_answer_nan(gpu, accumulate):
    """For their sequence alone; pages behind the length may name anything.  All of it is caught by bounds that the kernels check before they read."""
    import flex_block_attn_amd as fba

    lengths = [100, 100, 100, 100, 100, 0]
    cache, table, g = make(gpu, 6, 2, 128, 16)
    fill(cache, table, lengths, g)
    q = torch.randn((6, 4, 1, 128), generator=g).to(torch.bfloat16).to(gpu)
    good = check_attend(q, cache, table, lengths)
    weights = cache.weights.clone()
    table[0, 7:] = 1 << 30         # behind the length
    table[1, 3] = cache.k.shape[0]
    table[2, 0] = -1
    n = ints([100, 100, 100, 129, -1, 0], gpu)
    o = fba.cache_attn_func(q, cache, table, n, accumulate=accumulate)
    assert torch.equal(o[0], good[0]) and torch.equal(o[5], good[5])
    assert bool(o[1:5].isnan().all())
    if accumulate:
        for t in table[1:].reshape(-1).tolist():  # only the first sequence's weights have changed
            if 0 <= t < cache.k.shape[0]:
                assert torch.equal(cache.weights[t].nan_to_num(-5.0), weights[t].nan_to_num(-5.0))


def test_far_pages(gpu):
    """Offsets of rows in bytes that pass 32 bits."""
    import flex_block_attn_amd as fba

    pages, Hk, page = 70000, 8, 128
    cache = fba.paged_cache(pages, Hk, page, device=gpu, bits=4)
    assert (pages * Hk - 1) * page * 64 > 2**32
    near = fba.paged_cache(2, Hk, page, device=gpu, bits=4)
    table, near_table = ints([[pages - 1, pages - 2]], gpu), ints([[1, 0]], gpu)
    g = torch.Generator(device="cpu").manual_seed(2)
    k, v, q = (torch.randn((1, Hk, n, 128), generator=g).to(torch.bfloat16).to(gpu) for n in (200, 200, 1))
    turn = fba.rotary(device=gpu)
    zero = ints([0], gpu)
    n, _ = fba.cache_append_rotary(cache, table, zero, k, v, turn)
    fba.cache_append_rotary(near, near_table, zero, k, v, turn)
    for x, y in zip(fba.cache_read(cache, table, n, 200), fba.cache_read(near, near_table, n, 200)):
        assert torch.equal(x, y) and bool(x.any())
    assert torch.equal(fba.cache_attn_func(q, cache, table, n), fba.cache_attn_func(q, near, near_table, n))


# ---------------------------------------------------------------------------------------------------------------------
# eviction, and all of it together
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lengths,budget,recent,sinks,page", [
    ([1, 2, 0], 1, 0, 0, 16), ([100, 300, 64], 64, 64, 0, 16), ([1025, 1024, 2000], 1000, 30, 4, 64), ([5000, 4097], 4096, 256, 4, 32), ([2500, 10], 700, 0, 700, 256), ([33000, 32900], 32850, 100, 4, 64),
    ([1, 2, 3, 4, 5, 6, 7, 8], 1, 0, 0, 16), ([3000, 2048], 1, 1, 0, 128),
])
def test_evict(gpu, lengths, budget, recent, sinks, page):
    """The rows of the slots that change places, their scales with them."""
    import flex_block_attn_amd as fba

    cache, table, g = make(gpu, len(lengths), 2, max(lengths), page, seed=budget, extra=1)
    fill(cache, table, lengths, g)
    want = evict_reference(cache, table, lengths, budget, recent, sinks)
    scales = evict_reference(fba.PagedCache(cache.k_scales, cache.v_scales, cache.positions, cache.weights), table, lengths, budget, recent, sinks)
    print(f"evict {lengths} to {budget}, recent {recent}, sinks {sinks}, page {page}", flush=True)
    out = fba.cache_evict(cache, table, ints(lengths, gpu), budget, recent=recent, sinks=sinks)
    assert out.tolist() == [min(x, budget) for x in lengths]
    for name, x, y in zip(("k", "v", "positions", "weights", "k_scales", "v_scales"), (cache.k, cache.v, cache.positions, cache.weights, cache.k_scales, cache.v_scales), (*want, *scales[:2])):
        assert torch.equal(x.nan_to_num(-5.0) if x.is_floating_point() else x, y.nan_to_num(-5.0) if y.is_floating_point() else y), name


@pytest.mark.parametrize("bits", [4, 16])
def test_a_stream_with_positions(gpu, bits):
    """A prompt in two chunks, the second against what is read back, then tokens one by one: against a plain program that turns all keys by where they stand, holds them as the cache does, and
    attends in 64 bits."""
    import flex_block_attn_amd as fba

    B, H, Hk, page, S, chunk = 2, 6, 2, 16, 130, 50
    cache = fba.paged_cache(40, Hk, page, device=gpu, bits=bits)
    table = torch.arange(40, dtype=torch.int32, device=gpu).reshape(B, 20).flip(1).contiguous()
    g = torch.Generator(device="cpu").manual_seed(11)
    q, k, v = (torch.randn((B, h, S, 128), generator=g).to(torch.bfloat16).to(gpu) for h in (H, Hk, Hk))
    turn = fba.rotary(device=gpu, interleaved=False)
    stand = torch.arange(S)[None, :, None].expand(B, S, 1)
    turned, u = exact(k, turn, stand)[0], 2.0**-8
    if bits == 4:
        keys, values = held(turned, torch.bfloat16)[0].to(gpu), held(v.double().cpu(), torch.bfloat16)[0].to(gpu)
    else:
        keys, values = turned.to(torch.bfloat16).double().to(gpu), v.double()
    qs = exact(q, turn, stand)[0].to(gpu)
    outs = []
    n = torch.zeros(B, dtype=torch.int32, device=gpu)
    for first in (0, chunk):
        part = slice(first, first + chunk)
        n, tq = fba.cache_append_rotary(cache, table, n, k[:, :, part], v[:, :, part], turn, q=q[:, :, part])
        outs.append(fba.window_attn_func(tq, *fba.cache_read(cache, table, n, first + chunk), None))
    for t in range(2 * chunk, S):
        n, tq = fba.cache_append_rotary(cache, table, n, k[:, :, t:t + 1], v[:, :, t:t + 1], turn, q=q[:, :, t:t + 1])
        outs.append(fba.cache_attn_func(tq, cache, table, n))
    assert n.tolist() == [S, S]
    keys, values = (x.repeat_interleave(H // Hk, 1) for x in (keys, values))
    scores = qs @ keys.transpose(2, 3).contiguous() / math.sqrt(128)
    p = torch.softmax(scores.masked_fill(torch.ones(S, S, dtype=torch.bool, device=gpu).triu(1), -math.inf), -1)
    want = p @ values
    # q (and in 16 bits k) rounded after the rotation: every score is off by u |q| |k| of it, twice in 16 bits, so weights by twice that; P of a chunk and o rounded, u each
    most = u * (2 if bits == 16 else 1) * (qs.abs() @ keys.abs().transpose(2, 3).contiguous()).amax() / math.sqrt(128)
    off = ((2 * most).expm1() + 2 * u) * (p @ values.abs()) + u * want.abs() + 1e-6
    over = (torch.cat(outs, 2).double() - want).abs() - off
    assert bool((over <= 0).all()), f"{over.max().item():.3e} beyond the bound"


def test_a_stream_under_a_budget(gpu):
    """Tokens one by one into 4 bits, attended with weights added up, evicted to the budget: what is kept is what a plain program keeps."""
    import flex_block_attn_amd as fba

    B, H, Hk, page, budget, recent, sinks = 2, 4, 2, 16, 40, 8, 2
    cache, table, g = make(gpu, B, Hk, budget + 30, page)
    new = lambda n, h=Hk: torch.randn((B, h, n, 128), generator=g).to(torch.bfloat16).to(gpu)
    turn = fba.rotary(device=gpu)
    seen = ints([30, 55], gpu)
    lengths, _ = fba.cache_append_rotary(cache, table, torch.zeros_like(seen), new(55), new(55), turn, counts=seen)
    for _ in range(15):
        lengths, q = fba.cache_append_rotary(cache, table, lengths, new(1), new(1), turn, q=new(1, H), positions=seen)
        seen = seen + 1
        check_attend(q, cache, table, lengths.tolist(), accumulate=True)
        want = evict_reference(cache, table, lengths.tolist(), budget, recent, sinks)
        lengths = fba.cache_evict(cache, table, lengths, budget, recent=recent, sinks=sinks)
        for x, y in zip((cache.k, cache.v, cache.positions, cache.weights), want):
            assert torch.equal(x.nan_to_num(-5.0) if x.is_floating_point() else x, y.nan_to_num(-5.0) if y.is_floating_point() else y)
    assert lengths.tolist() == [40, 40]


@pytest.mark.parametrize("bits", [4, 16])
def test_replays_from_a_captured_graph(gpu, bits):
    """A whole step recorded: rotation and append, attention, rows read back, eviction, and the lengths brought on.  Beside an eager program on caches of its own."""
    import flex_block_attn_amd as fba

    B, H, Hk, page, budget = 3, 8, 2, 16, 70
    turn = fba.rotary((64,), device=gpu)
    sides = []
    for _ in range(2):
        cache, table, g = make(gpu, B, Hk, budget + 1, page, seed=9)
        fill(cache, table, [60, 70, 1], g)
        sides.append(dict(cache=cache if bits == 4 else wide(cache), table=table, lengths=ints([60, 70, 1], gpu), seen=ints([60, 90, 1], gpu),
                          q=torch.zeros((B, H, 1, 128), dtype=torch.bfloat16, device=gpu), k=torch.zeros((B, Hk, 1, 128), dtype=torch.bfloat16, device=gpu),
                          v=torch.zeros((B, Hk, 1, 128), dtype=torch.bfloat16, device=gpu)))

    def step(s):
        n, q = fba.cache_append_rotary(s["cache"], s["table"], s["lengths"], s["k"], s["v"], turn, q=s["q"], positions=s["seen"])
        o = fba.cache_attn_func(q, s["cache"], s["table"], n, accumulate=True)
        back = fba.cache_read(s["cache"], s["table"], n, 75)
        n = fba.cache_evict(s["cache"], s["table"], n, budget, recent=8, sinks=2)
        s["lengths"].copy_(n)
        s["seen"].add_(1)
        return (o, *back)

    eager, recorded = sides
    moving = lambda s: {**every(s["cache"]), "lengths": s["lengths"], "seen": s["seen"]}
    start = {name: t.clone() for name, t in moving(recorded).items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(recorded)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(recorded)
    for name, t in moving(recorded).items():
        t.copy_(start[name])
    for _ in range(5):
        for name, h in (("q", H), ("k", Hk), ("v", Hk)):
            new = torch.randn((B, h, 1, 128), generator=g).to(torch.bfloat16).to(gpu)
            eager[name].copy_(new)
            recorded[name].copy_(new)
        want = step(eager)
        torch.cuda.synchronize()
        for t in out:
            t.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y)
        for x, y in zip(moving(eager).values(), moving(recorded).values()):
            assert torch.equal(x.nan_to_num(-5.0) if x.is_floating_point() else x, y.nan_to_num(-5.0) if y.is_floating_point() else y)


def test_on_two_streams(gpu):
    import flex_block_attn_amd as fba

    lengths = [3000, 100, 0, 2000]
    cache, table, g = make(gpu, 4, 2, 3000, 32)
    fill(cache, table, lengths, g)
    n = ints(lengths, gpu)
    qs = [torch.randn((4, 8, 1, 128), generator=g).to(torch.bfloat16).to(gpu) for _ in range(2)]
    want = [fba.cache_attn_func(q, cache, table, n) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(4):
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(fba.cache_attn_func(q, cache, table, n))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])


def test_strided_queries(gpu):
    import flex_block_attn_amd as fba

    cache, table, g = make(gpu, 2, 2, 200, 16)
    fill(cache, table, [200, 90], g)
    n = ints([200, 90], gpu)
    three = torch.randn((2, 1, 3, 8, 128), generator=g).to(torch.bfloat16).to(gpu)
    odd = torch.randn((2 * 8 * 128 + 3,), generator=g).to(torch.bfloat16).to(gpu)[3:].view(2, 8, 1, 128)
    for q in (three[:, :, 1].transpose(1, 2), odd, three[:, :, 0, :1].transpose(1, 2).expand(2, 8, 1, 128)):
        assert torch.equal(fba.cache_attn_func(q, cache, table, n), fba.cache_attn_func(q.contiguous().clone(), cache, table, n))


def test_writes_raise_the_versions_of_what_they_write_to(gpu):
    import flex_block_attn_amd as fba

    cache, table, g = make(gpu, 2, 2, 64, 16)
    fill(cache, table, [40, 20], g)
    n, turn = ints([40, 20], gpu), fba.rotary(device=gpu)
    row = lambda h: torch.ones((2, h, 1, 128), dtype=torch.bfloat16, device=gpu)
    everything = set(every(cache))
    for call, written in ((lambda: fba.cache_append(cache, table, n, row(2), row(2)), everything), (lambda: fba.cache_append_rotary(cache, table, n, row(2), row(2), turn, q=row(4)), everything),
                          (lambda: fba.cache_attn_func(row(4), cache, table, n), set()), (lambda: fba.cache_attn_func(row(4), cache, table, n, accumulate=True), {"weights"}),
                          (lambda: fba.cache_read(cache, table, n, 9), set()), (lambda: fba.cache_evict(cache, table, n, 30), everything)):
        before = {x: t._version for x, t in every(cache).items()}
        call()
        for x, t in every(cache).items():
            assert (t._version > before[x]) == (x in written), x
