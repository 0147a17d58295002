"""The paged cache with tables that have room for far more than the sequences hold, as a server's have: eviction and attention choose by that room."""
import pytest
import torch

from test_gpu_cache import check_attend, evict_reference, fill, make

pytestmark = pytest.mark.gpu


def _wide(gpu, lengths, Hk, page, room, seed=0):
    """As `make`, with tables of `room` slots: what is behind a sequence's own pages names none, or anything."""
    cache, table, g = make(gpu, len(lengths), Hk, max(lengths), page, seed=seed)
    fill(cache, table, lengths, g)
    wide = torch.full((len(lengths), room // page), -1, dtype=torch.int32, device=gpu)
    wide[:, 1::2] = 1 << 30
    wide[:, :table.shape[1]] = table
    return cache, table, wide, g


@pytest.mark.parametrize("room", [4096, 8192, 8208, 32768, 32784, 131072])
@pytest.mark.parametrize("lengths,budget,recent,sinks", [([1030, 1025, 1024, 3], 1024, 16, 4), ([3000, 2500, 100], 1000, 50, 10), ([700, 1], 1, 0, 0)])
def test_evict(gpu, room, lengths, budget, recent, sinks):
    import flex_block_attn_amd as fba

    cache, table, wide, _ = _wide(gpu, lengths, 2, 16, room, seed=room)
    want = evict_reference(cache, table, lengths, budget, recent, sinks)
    n = torch.tensor(lengths, dtype=torch.int32, device=gpu)
    print(f"evict {lengths} to {budget} in room for {room}", flush=True)
    assert fba.cache_evict(cache, wide, n, budget, recent=recent, sinks=sinks).tolist() == [min(x, budget) for x in lengths]
    for x, y in zip((cache.k, cache.v, cache.positions, cache.weights), want):
        assert torch.equal(x.nan_to_num(-5.0), y.nan_to_num(-5.0))


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("room", [2048, 40000, 1 << 20])
def test_attend(gpu, accumulate, room):
    lengths = [700, 0, 33, 1999]
    cache, table, wide, g = _wide(gpu, lengths, 2, 16, room, seed=room)
    q = (torch.randn((len(lengths), 6, 1, 128), generator=g) * 2).to(torch.bfloat16).to(gpu)
    check_attend(q, cache, wide, lengths, accumulate=accumulate)
    if not accumulate:
        check_attend(q, cache, wide, lengths, window=100, sinks=20)


def test_append(gpu):
    import flex_block_attn_amd as fba

    lengths = [700, 0, 33]
    cache, table, wide, g = _wide(gpu, lengths, 2, 16, 1 << 20)
    new = torch.randn((3, 2, 3, 128), generator=g).to(torch.bfloat16).to(gpu)
    n = torch.tensor(lengths, dtype=torch.int32, device=gpu)
    assert fba.cache_append(cache, wide, n, new, new, counts=torch.tensor([3, 2, 1], dtype=torch.int32, device=gpu)).tolist() == [703, 2, 34]
    for b, (at, c) in enumerate(zip(lengths, (3, 2, 1))):
        for t in range(c):
            page = int(table[b, (at + t) // 16])
            assert torch.equal(cache.k[page, :, (at + t) % 16], new[b, :, t]) and torch.equal(cache.v[page, :, (at + t) % 16], new[b, :, t])
    # onto a page that the table does not have
    n = torch.tensor([704, 0, 33], dtype=torch.int32, device=gpu)
    assert fba.cache_append(cache, wide[:, :44].contiguous(), n, new, new).tolist() == [-1, 3, 36]
