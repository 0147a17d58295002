"""Attention over 4 bits where its shares are cut at their ends: far more sequences than the GPU has places, tables of a single page that is less than a tile.  Against 64 bits with the bound of
test_gpu_cache.py."""
import pytest
import torch

from test_gpu_cache import attend_reference
from test_gpu_cache4 import check_attend, fill, ints, make, wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths,H,Hk", [
    ([(37 * i) % 71 for i in range(1500)], 4, 2), ([1] * 1031, 2, 2), ([0] * 700 + [33] + [0] * 699 + [32, 0, 65], 3, 1), ([i % 2 for i in range(900)], 34, 2),
])
def test_more_sequences_than_places(gpu, lengths, H, Hk):
    cache, table, g = make(gpu, len(lengths), Hk, max(lengths), 16, seed=len(lengths))
    fill(cache, table, lengths, g)
    q = torch.randn((len(lengths), H, 1, 128), generator=g).to(torch.bfloat16).to(gpu)
    check_attend(q, cache, table, lengths, accumulate=True)
    check_attend(q, cache, table, lengths, window=20, sinks=3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths", [[16], [16, 3, 0, 15, 1], [7] * 70])
def test_tables_of_one_page(gpu, dtype, lengths):
    cache, table, g = make(gpu, len(lengths), 2, 16, 16, dtype, seed=sum(lengths))
    assert table.shape[1] == 1
    fill(cache, table, lengths, g)
    q = torch.randn((len(lengths), 6, 1, 128), generator=g).to(dtype).to(gpu)
    check_attend(q, cache, table, lengths, accumulate=True)
    check_attend(q, cache, table, lengths, window=2, sinks=1)


def test_wrong_lengths_among_many(gpu):
    """A sequence whose length makes no sense has no tiles: it answers no numbers, and all others what is theirs."""
    import flex_block_attn_amd as fba

    B = 900
    lengths = [(13 * i) % 50 for i in range(B)]
    cache, table, g = make(gpu, B, 2, 64, 16, seed=3)
    fill(cache, table, lengths, g)
    q = torch.randn((B, 4, 1, 128), generator=g).to(torch.bfloat16).to(gpu)
    want, off, _, _ = attend_reference(q, wide(cache), table, lengths, None, 0)
    wrong = [i % 7 == 3 for i in range(B)]
    o = fba.cache_attn_func(q, cache, table, ints([(-1 if i % 2 else 65) if w else n for i, (w, n) in enumerate(zip(wrong, lengths))], gpu))
    wrong = torch.tensor(wrong, device=gpu)
    assert bool(o[wrong].isnan().all()) and bool(((o.double() - want).abs() <= off)[~wrong].all())
