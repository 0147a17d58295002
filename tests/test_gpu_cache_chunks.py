"""A prompt's next chunk over rows read back, in both of its forms: sequences of one length in one call, whatever the chunk adds to each, and sequences of different lengths one by one.  Against
the formula in 64 bits over what the cache holds, with the bound of test_gpu_window.py for o."""
import pytest
import torch

from test_gpu_cache4 import held
from test_gpu_window import reference

pytestmark = pytest.mark.gpu


def prompt(gpu, bits, before, counts, tokens, H=4, Hk=2, page=16):
    """A cache with `before` slots of every sequence and the next chunk, appended; (cache, table, lengths, q of the chunk, all keys and values of every sequence as they are held)"""
    import flex_block_attn_amd as fba

    B, g = len(before), torch.Generator(device="cpu").manual_seed(sum(before) + tokens)
    cache = fba.paged_cache(B * 20, Hk, page, device=gpu, bits=bits)
    for t in (cache.k, cache.v):
        t.fill_(255 if bits == 4 else float("nan"))
    if bits == 4:
        cache.k_scales.fill_(255)
        cache.v_scales.fill_(255)
    table = torch.randperm(B * 20, generator=g).to(torch.int32).reshape(B, 20).to(gpu)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    new = lambda h, n: torch.randn((B, h, n, 128), generator=g).to(torch.bfloat16)
    lengths, parts = torch.zeros(B, dtype=torch.int32, device=gpu), []
    for n in (before, counts):
        most = max(max(n), 1) if n is before else tokens
        k, v = new(Hk, most), new(Hk, most)
        lengths = fba.cache_append(cache, table, lengths, k.to(gpu), v.to(gpu), counts=ints(n))
        parts.append((k, v))
    assert lengths.tolist() == [a + b for a, b in zip(before, counts)]
    holds = lambda x: (held(x.double(), torch.bfloat16)[0] if bits == 4 else x).to(torch.bfloat16).to(gpu)
    all_of = [tuple(torch.cat([holds(parts[0][i][b:b + 1, :, :before[b]]), holds(parts[1][i][b:b + 1, :, :counts[b]])], 2) for i in (0, 1)) for b in range(B)]
    return cache, table, lengths, (new(H, tokens).float() * 2).to(torch.bfloat16).to(gpu), all_of


def check(o, q, keys, values, window, sinks):
    want, off = reference(q, keys, values, torch.zeros_like(q), window, sinks, True, None)
    over = (o.double() - want[0]).abs() - off[0]
    assert o.shape == q.shape and bool((over <= 0).all()), f"{over.max().item():.3e} beyond the bound"


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 3)])
@pytest.mark.parametrize("before,counts,tokens", [([37, 37, 37], [20, 5, 0], 20), ([0, 0], [33, 32], 33), ([64], [7], 40), ([150, 150], [1, 50], 64)])
def test_sequences_of_one_length(gpu, bits, window, sinks, before, counts, tokens):
    """One call for all: `slots` is what every sequence had and all of the chunk's tokens, so that a query stands where its token does; those behind a sequence's count are nobody's."""
    import flex_block_attn_amd as fba

    cache, table, lengths, q, all_of = prompt(gpu, bits, before, counts, tokens)
    o = fba.window_attn_func(q, *fba.cache_read(cache, table, lengths, before[0] + tokens), window, sinks=sinks)
    for b, (keys, values) in enumerate(all_of):
        if counts[b]:
            check(o[b:b + 1, :, :counts[b]], q[b:b + 1, :, :counts[b]], keys, values, window, sinks)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 3)])
@pytest.mark.parametrize("before,counts,tokens", [([37, 0, 112], [20, 20, 20], 20), ([5, 64, 63, 1], [17, 1, 40, 33], 40)])
def test_sequences_of_different_lengths(gpu, bits, window, sinks, before, counts, tokens):
    """One by one: as many slots as the sequence has, and its own queries."""
    import flex_block_attn_amd as fba

    cache, table, lengths, q, all_of = prompt(gpu, bits, before, counts, tokens)
    for b, (keys, values) in enumerate(all_of):
        own = q[b:b + 1, :, :counts[b]]
        k, v = fba.cache_read(cache, table[b:b + 1], lengths[b:b + 1], before[b] + counts[b])
        assert torch.equal(k, keys) and torch.equal(v, values)
        check(fba.window_attn_func(own, k, v, window, sinks=sinks), own, keys, values, window, sinks)
