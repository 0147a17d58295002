"""Arguments of the paged cache's operators where the native call and the Python one have to say the same."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _cache(gpu):
    import flex_block_attn_amd as fba

    cache = fba.paged_cache(4, 2, 16, device=gpu, evicting=True)
    for t in (cache.k, cache.v, cache.positions, cache.weights):
        t.zero_()
    return cache, torch.arange(4, dtype=torch.int32, device=gpu).reshape(1, 4), torch.tensor([20], dtype=torch.int32, device=gpu)


@pytest.mark.parametrize("window", [1, 64, 2**31 - 2, 2**31 - 1, 2**31, 2**40])
def test_accumulate_takes_no_window_however_wide(gpu, window):
    import flex_block_attn_amd as fba

    cache, table, n = _cache(gpu)
    for q in (torch.zeros((1, 4, 1, 128), dtype=torch.bfloat16, device=gpu), torch.zeros((1, 4, 1, 129), dtype=torch.bfloat16, device=gpu)[..., 1:]):
        with pytest.raises(ValueError, match="window must be None"):
            fba.cache_attn_func(q, cache, table, n, window=window, accumulate=True)
        assert int(fba.cache_attn_func(q, cache, table, n, window=window).count_nonzero()) == 0
        assert int(fba.cache_attn_func(q, cache, table, n, accumulate=True).count_nonzero()) == 0
    assert float(cache.weights.sum()) == pytest.approx(2 * 2 * 2, abs=1e-5)  # two calls, two kv heads of two query heads


def test_more_tokens_than_a_call_may_append(gpu):
    """A tensor that repeats one row can be as long; the error says what is wrong with it."""
    import flex_block_attn_amd as fba
    from flex_block_attn_amd import _lib

    cache, table, n = _cache(gpu)
    rows = torch.zeros((1, 2, 1, 128), dtype=torch.bfloat16, device=gpu).expand(1, 2, (1 << 28) + 1, 128)
    with pytest.raises(_lib.FbaError, match="2\\^28 tokens"):
        fba.cache_append(cache, table, n, rows, rows)
