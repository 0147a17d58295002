"""The paged cache: append, attention of one new token, eviction by weight, and the three together, against plain implementations (attention in 64 bits).

Tolerances of attention.  u = eps / 2 of the type, f = 2^-24.  Scores are fp32 sums of 128 products, off by 130 f of the sum of their sizes; exp2, the denominator and the
joins add up to 64 f: e.  P goes into the second product in two parts, off by u^2 of it, and, where fp16 ends, by 2^-25 of the largest; o is rounded once:
  o        (2e + u^2) P|v| + 2^-25 |v| summed + u|o|
  weights  (2e + heads f) P summed over heads + 2f |weights|
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(128)


def make(gpu, B, Hk, most, page, dtype=torch.bfloat16, seed=0, spare=3, extra=0):
    """(cache with everything, table): pages dealt out of order, what is not filled is no number."""
    import flex_block_attn_amd as fba

    g = torch.Generator(device="cpu").manual_seed(seed)
    per = -(-most // page) + extra
    pages = B * per + spare
    cache = fba.paged_cache(pages, Hk, page, dtype=dtype, device=gpu, evicting=True)
    for t in (cache.k, cache.v, cache.weights):
        t.fill_(math.nan)
    cache.positions.fill_(-7)
    table = torch.randperm(pages, generator=g)[: B * per].to(torch.int32).reshape(B, per).to(gpu)
    return cache, table, g


def fill(cache, table, lengths, g):
    """Random rows, weights and positions in the filled slots of every sequence."""
    page = cache.k.shape[2]
    for b, n in enumerate(lengths):
        for i in range(-(-max(0, n) // page)):
            m, at = min(page, n - i * page), int(table[b, i])
            shape = (cache.k.shape[1], m)
            cache.k[at, :, :m] = torch.randn((*shape, 128), generator=g).to(cache.k)
            cache.v[at, :, :m] = torch.randn((*shape, 128), generator=g).to(cache.v)
            cache.weights[at, :, :m] = (torch.rand(shape, generator=g) * 3).to(cache.weights)
            cache.positions[at, :, :m] = torch.arange(i * page, i * page + m, dtype=torch.int32).to(cache.positions)


def rows(t, table, b, n):
    """The first n slots of sequence b: (kv heads, n, ...)."""
    page = t.shape[2]
    s = torch.arange(n, device=t.device)
    return t[table[b].long()[s // page], :, s % page].transpose(0, 1)


def attend_reference(q, cache, table, lengths, window, sinks):
    """o, its bound; the weights that are added [b][kv heads, n], their bounds."""
    u, f = torch.finfo(q.dtype).eps / 2, 2.0**-24
    B, H = q.shape[:2]
    Hk = cache.k.shape[1]
    o, off, added, added_off = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device), [], []
    for b, n in enumerate(lengths):
        k, v = rows(cache.k, table, b, n).double(), rows(cache.v, table, b, n).double()
        s = torch.arange(n, device=q.device)
        seen = torch.ones_like(s, dtype=torch.bool) if window is None else (s >= n - window) | (s < sinks)
        k, v = k[:, seen], v[:, seen]
        qb = q[b, :, 0].double().reshape(Hk, H // Hk, 128)
        p = torch.softmax(qb @ k.transpose(1, 2).contiguous() * SCALE, -1)
        e = (130 * f * (qb.abs() @ k.abs().transpose(1, 2).contiguous()).max().item() * SCALE if n else 0.0) + 64 * f
        y = p @ v
        o[b, :, 0] = y.reshape(H, 128)
        off[b, :, 0] = ((2 * e + u * u) * (p @ v.abs()) + 2.0**-25 * v.abs().sum(1, keepdim=True) + u * y.abs()).reshape(H, 128)
        added.append(p.sum(1))
        added_off.append((2 * e + H // Hk * f) * p.sum(1))
    return o, off, added, added_off


def check_attend(q, cache, table, lengths, window=None, sinks=0, accumulate=False):
    import flex_block_attn_amd as fba

    print(f"attend q{tuple(q.shape)} cache{tuple(cache.k.shape)} table{tuple(table.shape)} lengths {lengths[:8]} window {window} sinks {sinks} accumulate {accumulate} {q.dtype}", flush=True)
    n = torch.tensor(lengths, dtype=torch.int32, device=q.device)
    want, off, added, added_off = attend_reference(q, cache, table, lengths, window, sinks)
    before = cache.weights.clone()
    o = fba.cache_attn_func(q, cache, table, n, window=window, sinks=sinks, accumulate=accumulate)
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
    """Slots between the sinks and the window hold infinities here: they are not seen."""
    lengths = [0, 1, 31, 64, 100, 333, 1500]
    cache, table, g = make(gpu, len(lengths), 2, max(lengths), 16, seed=window)
    fill(cache, table, lengths, g)
    for b, n in enumerate(lengths):
        for s in range(sinks, max(sinks, n - window)):
            at = int(table[b, s // 16])
            cache.k[at, :, s % 16] = math.inf if s % 3 else math.nan
            cache.v[at, :, s % 16] = math.nan if s % 2 else -math.inf
    q = (torch.randn((len(lengths), 6, 1, 128), generator=g) * 2).to(torch.bfloat16).to(gpu)
    check_attend(q, cache, table, lengths, window=window, sinks=sinks)


@pytest.mark.parametrize("B", [63, 64, 65, 200])
def test_attend_many_sequences(gpu, B):
    lengths = [(37 * i) % 211 for i in range(B)]
    cache, table, g = make(gpu, B, 2, max(lengths), 16, seed=B)
    fill(cache, table, lengths, g)
    q = torch.randn((B, 4, 1, 128), generator=g).to(torch.bfloat16).to(gpu)
    check_attend(q, cache, table, lengths, accumulate=True)


def test_attend_far_pages_and_large_scores(gpu):
    """Rows whose offsets pass 31 bits, and scores so large that one slot has all the weight."""
    import flex_block_attn_amd as fba

    pages, Hk, page = 9000, 8, 128
    cache = fba.PagedCache(*(torch.empty((pages, Hk, page, 128), dtype=torch.bfloat16, device=gpu) for _ in range(2)),
                           positions=torch.empty((pages, Hk, page), dtype=torch.int32, device=gpu), weights=torch.zeros((pages, Hk, page), device=gpu))
    last = (pages * Hk - 1) * page * 128 * 2  # bytes in front of the last page's last head
    assert last > 2**31
    table = torch.tensor([[8999, 0, 8998], [8997, 8996, 1]], dtype=torch.int32, device=gpu)
    g = torch.Generator(device="cpu").manual_seed(1)
    new = lambda n: torch.randn((2, Hk, n, 128), generator=g).to(torch.bfloat16).to(gpu)
    lengths = torch.zeros(2, dtype=torch.int32, device=gpu)
    k, v = new(300), new(300)
    lengths = fba.cache_append(cache, table, lengths, k, v)
    assert lengths.tolist() == [300, 300]
    assert torch.equal(rows(cache.k, table, 0, 300), k[0]) and torch.equal(rows(cache.v, table, 1, 300), v[1])
    q = torch.randn((2, 8, 1, 128), generator=g).to(torch.bfloat16).to(gpu)
    check_attend(q, cache, table, [300, 300], accumulate=True)
    check_attend(q * 300, cache, table, [300, 300], accumulate=True)


def test_attend_very_far_page(gpu):
    """A pool of 5 GB: a row's offset in bytes passes 32 bits."""
    import flex_block_attn_amd as fba

    pages, Hk, page = 19600, 8, 128
    cache = fba.PagedCache(*(torch.empty((pages, Hk, page, 128), dtype=torch.bfloat16, device=gpu) for _ in range(2)))
    last = (pages * Hk - 1) * page * 128 * 2
    assert last > 2**32
    table = torch.tensor([[19599, 19598]], dtype=torch.int32, device=gpu)
    g = torch.Generator(device="cpu").manual_seed(2)
    k, v = (torch.randn((1, Hk, 200, 128), generator=g).to(torch.bfloat16).to(gpu) for _ in range(2))
    n = fba.cache_append(cache, table, torch.zeros(1, dtype=torch.int32, device=gpu), k, v)
    q = torch.randn((1, 8, 1, 128), generator=g).to(torch.bfloat16).to(gpu)
    near = fba.PagedCache(*(t.reshape(Hk, 200, 128)[None].contiguous().new_zeros((2, Hk, 128, 128)) for t in (k, v)))
    near_table = torch.tensor([[1, 0]], dtype=torch.int32, device=gpu)
    fba.cache_append(near, near_table, torch.zeros(1, dtype=torch.int32, device=gpu), k, v)
    assert torch.equal(fba.cache_attn_func(q, cache, table, n), fba.cache_attn_func(q, near, near_table, n))


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
    n = torch.tensor([100, 100, 100, 129, -1, 0], dtype=torch.int32, device=gpu)
    o = fba.cache_attn_func(q, cache, table, n, accumulate=accumulate)
    assert torch.equal(o[0], good[0]) and torch.equal(o[5], good[5])
    assert bool(o[1:5].isnan().all())
    if not accumulate:
        return
    for t in table[1:].reshape(-1).tolist():  # only the first sequence's weights have changed
        if 0 <= t < cache.k.shape[0]:
            assert torch.equal(cache.weights[t].nan_to_num(-5.0), weights[t].nan_to_num(-5.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,before,counts", [(16, [0, 5, 16, 40], [1, 1, 1, 1]), (16, [0, 5, 16, 40], [37, 0, 16, 3]), (64, [63, 64, 65], [200, 129, 1]), (256, [10], [1000])])
def test_append(gpu, dtype, page, before, counts):
    import flex_block_attn_amd as fba

    B, Hk, T = len(before), 3, max(counts)
    cache, table, g = make(gpu, B, Hk, max(a + c for a, c in zip(before, counts)), page, dtype)
    fill(cache, table, before, g)
    want = [t.clone() for t in (cache.k, cache.v, cache.positions, cache.weights)]
    k, v = (torch.randn((B, T, Hk, 128), generator=g).to(dtype).to(gpu).transpose(1, 2) for _ in range(2))
    first = torch.tensor([1000 * b for b in range(B)], dtype=torch.int32, device=gpu)
    weights = torch.rand((B, Hk, T), generator=g).to(gpu)
    n, c = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in (before, counts))
    out = fba.cache_append(cache, table, n, k, v, counts=c, positions=first, weights=weights)
    assert out.tolist() == [a + x for a, x in zip(before, counts)] and n.tolist() == before and out.data_ptr() != n.data_ptr()
    for b in range(B):
        for t in range(counts[b]):
            at, s = int(table[b, (before[b] + t) // page]), (before[b] + t) % page
            want[0][at, :, s], want[1][at, :, s] = k[b, :, t], v[b, :, t]
            want[2][at, :, s], want[3][at, :, s] = 1000 * b + t, weights[b, :, t]
    for x, y in zip((cache.k, cache.v, cache.positions, cache.weights), want):
        assert torch.equal(x.nan_to_num(-5.0), y.nan_to_num(-5.0))
    # without counts, positions and weights: all of them, at the slots' positions, with nothing yet
    if counts == [T] * B:
        again = fba.cache_append(cache, table, n, k, v)
        assert torch.equal(again, out)
        for b in range(B):
            assert torch.equal(rows(cache.positions, table, b, before[b] + T)[:, before[b]:], torch.arange(before[b], before[b] + T, dtype=torch.int32, device=gpu).expand(Hk, T))
            assert int(rows(cache.weights, table, b, before[b] + T)[:, before[b]:].count_nonzero()) == 0


def test_append_where_there_is_no_room(gpu):
    """Lengths, counts and pages that make no sense are answered with -1: nothing is written but rows on good pages of a table with a bad one."""
    import flex_block_attn_amd as fba

    cache, table, g = make(gpu, 6, 2, 64, 16)
    table[4, 1] = -3
    before = [t.clone() for t in (cache.k, cache.v, cache.positions, cache.weights)]
    k, v = (torch.randn((6, 2, 20, 128), generator=g).to(torch.bfloat16).to(gpu) for _ in range(2))
    n = torch.tensor([45, 65, -1, 10, 10, 44], dtype=torch.int32, device=gpu)
    c = torch.tensor([20, 1, 1, 21, 20, 20], dtype=torch.int32, device=gpu)
    out = fba.cache_append(cache, table, n, k, v, counts=c)
    assert out.tolist() == [-1, -1, -1, -1, -1, 64]
    for t in (0, 1, 2, 3):
        for p in table[t].tolist():
            for x, y in zip((cache.k, cache.v, cache.positions, cache.weights), before):
                assert torch.equal(x[p].nan_to_num(-5.0), y[p].nan_to_num(-5.0))
    assert torch.equal(rows(cache.k, table, 5, 64)[:, 44:], k[5])
    # what -1 is handed on to stays -1
    assert fba.cache_append(cache, table, out, k, v).tolist()[:5] == [-1] * 5
    assert fba.cache_evict(cache, table, out, 40).tolist() == [-1] * 5 + [40]


def evict_reference(cache, table, lengths, budget, recent, sinks):
    k, v, positions, weights = (t.clone() for t in (cache.k, cache.v, cache.positions, cache.weights))
    page = k.shape[2]
    tables, at, w = table.tolist(), positions.tolist(), weights.tolist()
    for b, n in enumerate(lengths):
        if n <= budget:
            continue
        place = [(tables[b][s // page], s % page) for s in range(n)]
        for h in range(k.shape[1]):
            newest = max(at[p][h][s] for p, s in place)

            def order(slot):
                p, s = place[slot]
                held = at[p][h][s] < sinks or at[p][h][s] > newest - recent
                weight = w[p][h][s]
                return (0 if held else 1, 0 if held else (math.inf if math.isnan(weight) else -weight), 1 if not held and math.isnan(weight) else 0, slot)

            kept = set(sorted(range(n), key=order)[:budget])
            free, late = [s for s in range(budget) if s not in kept], [s for s in range(budget, n) if s in kept]
            assert len(free) == len(late)
            if not free:
                continue
            to, source = (torch.tensor([place[s] for s in x]).to(k.device).unbind(1) for x in (free, late))
            for t in (k, v, positions, weights):
                t[to[0], h, to[1]] = t[source[0], h, source[1]]
    return k, v, positions, weights


@pytest.mark.parametrize("kind", ["random", "ties", "equal", "signs"])
@pytest.mark.parametrize("lengths,budget,recent,sinks,page", [
    ([1, 2, 0], 1, 0, 0, 16), ([33, 32, 31], 32, 4, 2, 16), ([100, 300, 64], 64, 64, 0, 16), ([1025, 1024, 2000], 1000, 30, 4, 64), ([3000, 2048], 1, 1, 0, 128),
    ([5000, 4097], 4096, 256, 4, 32), ([2500, 10], 700, 0, 700, 256), ([40000], 9000, 100, 10, 256),
    (list(range(40, 50)), 40, 5, 2, 16), (list(range(1020, 1032)), 1022, 1000, 22, 64), ([1, 2, 3, 4, 5, 6, 7, 8], 1, 0, 0, 16), ([12293, 12290, 12289], 12288, 64, 4, 128), ([33000, 32900], 32850, 100, 4, 64),
])
def test_evict(gpu, kind, lengths, budget, recent, sinks, page):
    import flex_block_attn_amd as fba

    cache, table, g = make(gpu, len(lengths), 2, max(lengths), page, seed=budget, extra=1)
    fill(cache, table, lengths, g)
    for b, n in enumerate(lengths):  # slots in no order, each head for itself
        for h in range(2):
            s, at = torch.arange(n, device=gpu), torch.randperm(n, generator=g).to(gpu) * 3
            cache.positions[table[b].long()[s // page], h, s % page] = at.to(torch.int32)
    w = cache.weights
    if kind == "ties":
        w.copy_((w * 3).floor())
    elif kind == "equal":
        w.copy_(torch.where(w.isnan(), w, torch.ones_like(w)))
    elif kind == "signs":  # weights that a program has set: both zeros, negative ones, infinities and no numbers
        values = torch.tensor([0.0, -0.0, -1.0, 1e-42, -1e-42, math.inf, -math.inf, math.nan, 2.5, 1e30], device=gpu)
        w.copy_(torch.where(w.isnan(), w, values[torch.randint(0, 10, w.shape, generator=g).to(gpu)]))
    want = evict_reference(cache, table, lengths, budget, recent, sinks)
    n = torch.tensor(lengths, dtype=torch.int32, device=gpu)
    print(f"evict {lengths} to {budget}, recent {recent}, sinks {sinks}, page {page}, {kind}", flush=True)
    out = fba.cache_evict(cache, table, n, budget, recent=recent, sinks=sinks)
    assert out.tolist() == [min(x, budget) for x in lengths] and n.tolist() == lengths
    for name, x, y in zip(("k", "v", "positions", "weights"), (cache.k, cache.v, cache.positions, cache.weights), want):
        assert torch.equal(x.view(torch.int16) if x.dtype == torch.bfloat16 else x.view(torch.int32), y.view(torch.int16) if y.dtype == torch.bfloat16 else y.view(torch.int32)), name
    again = fba.cache_evict(cache, table, out, budget, recent=recent, sinks=sinks)  # nothing is left to do
    assert torch.equal(again, out)
    for x, y in zip((cache.k, cache.v, cache.positions, cache.weights), want):
        assert torch.equal(x.view(torch.int16) if x.dtype == torch.bfloat16 else x.view(torch.int32), y.view(torch.int16) if y.dtype == torch.bfloat16 else y.view(torch.int32))


def test_evict_with_a_budget_beyond_the_table(gpu):
    import flex_block_attn_amd as fba

    cache, table, g = make(gpu, 2, 1, 64, 16)
    fill(cache, table, [64, 20], g)
    before = cache.weights.clone()
    n = torch.tensor([64, 20], dtype=torch.int32, device=gpu)
    assert fba.cache_evict(cache, table, n, 1000, recent=500, sinks=500).tolist() == [64, 20]
    assert torch.equal(before.nan_to_num(-5.0), cache.weights.nan_to_num(-5.0))


def test_a_stream_under_a_budget(gpu):
    """Prompt, then tokens one by one: appended, attended with weights added up, evicted to the budget.  What is attended to is what a plain program keeps, which takes the
    weights as the cache has them (two that differ by less than rounding could go either way)."""
    import flex_block_attn_amd as fba

    B, H, Hk, page, budget, recent, sinks = 3, 8, 2, 16, 60, 10, 2
    cache, table, g = make(gpu, B, Hk, budget + 40, page)
    new = lambda n: torch.randn((B, Hk, n, 128), generator=g).to(torch.bfloat16).to(gpu)
    lengths = torch.zeros(B, dtype=torch.int32, device=gpu)
    seen = torch.tensor([50, 80, 7], dtype=torch.int32, device=gpu)
    prompt = new(80)
    lengths = fba.cache_append(cache, table, lengths, prompt, new(80), counts=seen)
    for step in range(30):
        lengths = fba.cache_append(cache, table, lengths, new(1), new(1), positions=seen)
        seen = seen + 1
        q = (torch.randn((B, H, 1, 128), generator=g) * 2).to(torch.bfloat16).to(gpu)
        check_attend(q, cache, table, lengths.tolist(), accumulate=True)
        want = evict_reference(cache, table, lengths.tolist(), budget, recent, sinks)
        lengths = fba.cache_evict(cache, table, lengths, budget, recent=recent, sinks=sinks)
        for x, y in zip((cache.k, cache.v, cache.positions, cache.weights), want):
            assert torch.equal(x.nan_to_num(-5.0), y.nan_to_num(-5.0))
    assert lengths.tolist() == [60, 60, 37]
    for b in range(B):  # the last tokens and the first are there
        n = int(lengths[b])
        at = rows(cache.positions, table, b, n)
        for h in range(Hk):
            have = set(at[h].tolist())
            assert len(have) == n and set(range(sinks)) <= have and set(range(int(seen[b]) - recent, int(seen[b]))) <= have


def test_prefill_in_windows_then_tokens_one_by_one(gpu):
    """The last row of window_attn_func over n tokens and cache_attn_func over the same n say the same."""
    import flex_block_attn_amd as fba

    B, H, Hk, S, window, sinks = 2, 6, 2, 300, 70, 5
    cache, table, g = make(gpu, B, Hk, S, 32)
    q, k, v = (torch.randn((B, h, S, 128), generator=g).to(torch.bfloat16).to(gpu) for h in (H, Hk, Hk))
    o = fba.window_attn_func(q, k, v, window, sinks=sinks)
    lengths = fba.cache_append(cache, table, torch.zeros(B, dtype=torch.int32, device=gpu), k[:, :, :250], v[:, :, :250])
    for t in range(250, S):
        lengths = fba.cache_append(cache, table, lengths, k[:, :, t:t + 1], v[:, :, t:t + 1])
        one = fba.cache_attn_func(q[:, :, t:t + 1], cache, table, lengths, window=window, sinks=sinks)
        # both are within their bounds of the exact value: P rounded to bf16 (2^-7 of |v| <= 6 weighed), and o, twice
        assert float((one.double() - o[:, :, t:t + 1].double()).abs().max()) <= 2.0**-7 * 6


def test_replays_from_a_captured_graph(gpu):
    """A whole step recorded: append, attention, eviction, and the lengths brought on.  Beside an eager program on caches of its own."""
    import flex_block_attn_amd as fba

    B, H, Hk, page, budget = 3, 8, 2, 16, 70
    sides = []
    for _ in range(2):
        cache, table, g = make(gpu, B, Hk, budget + 1, page, seed=9)
        fill(cache, table, [60, 70, 1], g)
        sides.append(dict(cache=cache, table=table, lengths=torch.tensor([60, 70, 1], dtype=torch.int32, device=gpu), seen=torch.tensor([60, 90, 1], dtype=torch.int32, device=gpu),
                          q=torch.zeros((B, H, 1, 128), dtype=torch.bfloat16, device=gpu), k=torch.zeros((B, Hk, 1, 128), dtype=torch.bfloat16, device=gpu),
                          v=torch.zeros((B, Hk, 1, 128), dtype=torch.bfloat16, device=gpu)))

    def step(s):
        n = fba.cache_append(s["cache"], s["table"], s["lengths"], s["k"], s["v"], positions=s["seen"])
        o = fba.cache_attn_func(s["q"], s["cache"], s["table"], n, accumulate=True)
        n = fba.cache_evict(s["cache"], s["table"], n, budget, recent=8, sinks=2)
        s["lengths"].copy_(n)
        s["seen"].add_(1)
        return o

    eager, recorded = sides
    start = {name: t.clone() for name, t in (("k", recorded["cache"].k), ("v", recorded["cache"].v), ("p", recorded["cache"].positions), ("w", recorded["cache"].weights),
                                             ("n", recorded["lengths"]), ("s", recorded["seen"]))}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(recorded)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(recorded)
    for name, t in (("k", recorded["cache"].k), ("v", recorded["cache"].v), ("p", recorded["cache"].positions), ("w", recorded["cache"].weights), ("n", recorded["lengths"]), ("s", recorded["seen"])):
        t.copy_(start[name])
    for _ in range(5):
        for name, h in (("q", H), ("k", Hk), ("v", Hk)):
            new = torch.randn((B, h, 1, 128), generator=g).to(torch.bfloat16).to(gpu)
            eager[name].copy_(new)
            recorded[name].copy_(new)
        want = step(eager)
        torch.cuda.synchronize()
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(eager["lengths"], recorded["lengths"])
        for x, y in zip(vars(eager["cache"]).values(), vars(recorded["cache"]).values()):
            assert torch.equal(x.nan_to_num(-5.0), y.nan_to_num(-5.0))


def test_on_another_stream_and_beside_another_call(gpu):
    import flex_block_attn_amd as fba

    lengths = [3000, 100, 0, 2000]
    cache, table, g = make(gpu, 4, 2, 3000, 32)
    fill(cache, table, lengths, g)
    n = torch.tensor(lengths, dtype=torch.int32, device=gpu)
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


def test_strided_queries_and_rows(gpu):
    import flex_block_attn_amd as fba

    cache, table, g = make(gpu, 2, 2, 200, 16)
    fill(cache, table, [200, 90], g)
    n = torch.tensor([200, 90], dtype=torch.int32, device=gpu)
    wide = torch.randn((2, 1, 3, 8, 128), generator=g).to(torch.bfloat16).to(gpu)
    odd = torch.randn((2 * 8 * 128 + 3,), generator=g).to(torch.bfloat16).to(gpu)[3:].view(2, 8, 1, 128)
    for q in (wide[:, :, 1].transpose(1, 2), odd, wide[:, :, 0, :1].transpose(1, 2).expand(2, 8, 1, 128)):
        assert torch.equal(fba.cache_attn_func(q, cache, table, n), fba.cache_attn_func(q.contiguous().clone(), cache, table, n))
    rows_ = torch.randn((2, 2, 5, 129), generator=g).to(torch.bfloat16).to(gpu)[..., 1:]
    small = torch.tensor([10, 20], dtype=torch.int32, device=gpu)
    fba.cache_append(cache, table, small, rows_, rows_)
    assert torch.equal(rows(cache.k, table, 1, 25)[:, 20:], rows_[1])


def test_append_of_nothing(gpu):
    import flex_block_attn_amd as fba

    cache, table, g = make(gpu, 5, 2, 64, 16)
    n = torch.tensor([0, 64, 65, -2, 3], dtype=torch.int32, device=gpu)
    k = torch.empty((5, 2, 0, 128), dtype=torch.bfloat16, device=gpu)
    assert fba.cache_append(cache, table, n, k, k).tolist() == [0, 64, -1, -1, 3]
    assert fba.cache_append(cache, table, n, k, k, counts=torch.tensor([0, 0, 0, 0, 1], dtype=torch.int32, device=gpu)).tolist() == [0, 64, -1, -1, -1]


def test_pages_that_several_sequences_read(gpu):
    """A prompt that all share stands in the table of each: only what is written to may not."""
    import flex_block_attn_amd as fba

    cache, table, g = make(gpu, 3, 2, 200, 16)
    fill(cache, table, [200, 200, 200], g)
    shared = table.clone()
    shared[1:, :5] = table[0, :5]
    lengths = [200, 120, 81]
    q = torch.randn((3, 4, 1, 128), generator=g).to(torch.bfloat16).to(gpu)
    check_attend(q, cache, shared, lengths)
    check_attend(q, cache, shared, lengths, window=50, sinks=20)
    n = torch.tensor([200, 80, 80], dtype=torch.int32, device=gpu)
    k = torch.randn((3, 2, 1, 128), generator=g).to(torch.bfloat16).to(gpu)
    n = fba.cache_append(cache, torch.cat([shared, table[:, :1]], 1).contiguous(), n, k, k, counts=torch.tensor([0, 1, 1], dtype=torch.int32, device=gpu))
    assert n.tolist() == [200, 81, 81] and torch.equal(rows(cache.k, shared, 2, 81)[:, 80:], k[2])


def test_graphs_that_replay_in_turn_on_two_streams(gpu):
    """Each has a workspace of its own."""
    import flex_block_attn_amd as fba

    lengths = [2000, 100, 0, 900]
    cache, table, g = make(gpu, 4, 2, 2000, 32)
    fill(cache, table, lengths, g)
    n = torch.tensor(lengths, dtype=torch.int32, device=gpu)
    qs = [torch.randn((4, 8, 1, 128), generator=g).to(torch.bfloat16).to(gpu) for _ in range(2)]
    want = [fba.cache_attn_func(q, cache, table, n) for q in qs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in qs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(fba.cache_attn_func(q, cache, table, n))
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(4):
        for o in outs:
            o.fill_(math.nan)
        for s, graph in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
