"""The paged cache inside of programs that differentiate through its tensors: what the cache's operators write to counts as written."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _cache(gpu, evicting=True):
    import flex_block_attn_amd as fba

    cache = fba.paged_cache(6, 2, 16, device=gpu, evicting=evicting)
    for t in (cache.k, cache.v, cache.positions, cache.weights):
        if t is not None:
            t.zero_()
    table = torch.arange(6, dtype=torch.int32, device=gpu).reshape(2, 3)
    return cache, table, torch.tensor([40, 20], dtype=torch.int32, device=gpu)


def _calls():
    import flex_block_attn_amd as fba

    row = lambda gpu, h: torch.ones((2, h, 1, 128), dtype=torch.bfloat16, device=gpu)
    odd = lambda gpu, h: torch.ones((2, h, 1, 129), dtype=torch.bfloat16, device=gpu)[..., 1:]  # what Python prepares
    return {
        "append": (lambda gpu, c, t, n: fba.cache_append(c, t, n, row(gpu, 2), row(gpu, 2)), {"k", "v", "positions", "weights"}),
        "append of unaligned rows": (lambda gpu, c, t, n: fba.cache_append(c, t, n, odd(gpu, 2), odd(gpu, 2)), {"k", "v", "positions", "weights"}),
        "attention": (lambda gpu, c, t, n: fba.cache_attn_func(row(gpu, 4), c, t, n), set()),
        "attention with weights": (lambda gpu, c, t, n: fba.cache_attn_func(row(gpu, 4), c, t, n, accumulate=True), {"weights"}),
        "eviction": (lambda gpu, c, t, n: fba.cache_evict(c, t, n, 30), {"k", "v", "positions", "weights"}),
    }


@pytest.mark.parametrize("name", ["append", "append of unaligned rows", "attention", "attention with weights", "eviction"])
def test_writes_raise_the_versions_of_what_they_write_to(gpu, name):
    call, written = _calls()[name]
    cache, table, n = _cache(gpu)
    before = {x: t._version for x, t in vars(cache).items()}
    call(gpu, cache, table, n)
    for x, t in vars(cache).items():
        assert (t._version > before[x]) == (x in written), x
    if "weights" in written and "k" in written and name != "eviction":  # without what the cache does not have
        import flex_block_attn_amd as fba

        call(gpu, fba.PagedCache(cache.k, cache.v), table, n)


@pytest.mark.parametrize("field", ["k", "v", "weights"])
def test_backward_of_what_saved_the_cache_raises_after_eviction(gpu, field):
    """As it does for any operation in place, also where the saved tensor is a view of the cache's."""
    import flex_block_attn_amd as fba

    cache, table, n = _cache(gpu)
    x = torch.ones((2, 16, 1), device=gpu, requires_grad=True)
    t = getattr(cache, field)
    saved = t if field == "weights" else t[1:]
    y = (x.to(saved.dtype).reshape(2, 16, *[1] * (saved.dim() - 3)) * saved).sum()
    fba.cache_evict(cache, table, n, 30)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_caches_made_in_inference_mode(gpu):
    """Such tensors have no versions; they are taken inside of that mode and outside of it, as before."""
    import flex_block_attn_amd as fba

    with torch.inference_mode():
        cache, table, n = _cache(gpu)
        row = torch.ones((2, 2, 1, 128), dtype=torch.bfloat16, device=gpu)
        n = fba.cache_append(cache, table, n, row, row)
        o = fba.cache_attn_func(torch.ones((2, 4, 1, 128), dtype=torch.bfloat16, device=gpu), cache, table, n, accumulate=True)
        assert fba.cache_evict(cache, table, n, 30).tolist() == [30, 21] and bool(torch.isfinite(o).all())
    with torch.no_grad():
        assert fba.cache_append(cache, table, n, row, row).tolist() == [42, 22]
        assert fba.cache_evict(cache, table, n, 30).tolist() == [30, 21]
