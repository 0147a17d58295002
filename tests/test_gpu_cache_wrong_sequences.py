"""What a sequence with a wrong page does to others of its batch: nothing."""
import pytest
import torch

from test_gpu_cache import fill, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths", [[100, 100], [3000, 3000], [5000, 700]])
def test_weights_of_pages_that_a_wrong_sequence_names(gpu, lengths):
    """A sequence that is answered NaN writes nothing, so that it may name pages that another one adds weights to (a row of the table that is out of date)."""
    import flex_block_attn_amd as fba

    page = 16
    n = torch.tensor(lengths, dtype=torch.int32, device=gpu)
    results = []
    for shared in (False, True):
        cache, table, g = make(gpu, 2, 2, max(lengths), page, seed=5)
        fill(cache, table, lengths, g)
        own = table.clone()
        if shared:
            table[1] = table[0]
        table[1, (min(lengths) - 1) // page] = cache.k.shape[0]
        q = torch.randn((2, 8, 1, 128), generator=g).to(torch.bfloat16).to(gpu)
        before = cache.weights.clone()
        for _ in range(5):
            o = fba.cache_attn_func(q, cache, table, n, accumulate=True)
            assert bool(o[1].isnan().all())
        for p in own[1].tolist():  # the second one's own pages
            assert torch.equal(cache.weights[p].nan_to_num(-5.0), before[p].nan_to_num(-5.0))
        results.append((o[0], cache.weights[own[0].long()].nan_to_num(-5.0)))
    for x, y in zip(*results):
        assert torch.equal(x, y)
