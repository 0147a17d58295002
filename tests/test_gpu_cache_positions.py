"""Attention has no use for a cache's positions: whatever stands there is not looked at, on any path; what fills and evicts refuses it."""
from dataclasses import replace

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
def test_attention_does_not_look_at_positions(gpu, bits):
    import flex_block_attn_amd as fba

    cache = fba.paged_cache(4, 2, 16, device=gpu, evicting=True, bits=bits)
    g = torch.Generator(device="cpu").manual_seed(1)
    table, n = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32, device=gpu), torch.zeros(2, dtype=torch.int32, device=gpu)
    q, k, v = (torch.randn((2, h, m, 128), generator=g).to(torch.bfloat16).to(gpu) for h, m in ((4, 1), (2, 20), (2, 20)))
    n = fba.cache_append(cache, table, n, k, v)
    odd = torch.nn.functional.pad(q, (1, 0))[..., 1:]  # rows that Python prepares
    p = cache.positions
    for other in (None, p.long(), p.cpu(), p[:2], p.transpose(0, 1), torch.zeros(p.numel() + 1, dtype=torch.int32, device=gpu)[1:].view(p.shape), p.tolist()):
        some = replace(cache, positions=other)
        for accumulate in (False, True):
            cache.weights.zero_()
            want, added = fba.cache_attn_func(q, cache, table, n, accumulate=accumulate), cache.weights.clone()
            for x in (q, odd):
                cache.weights.zero_()
                assert torch.equal(fba.cache_attn_func(x, some, table, n, accumulate=accumulate), want) and torch.equal(cache.weights, added)
        if other is not None:
            for call in (lambda: fba.cache_append(some, table, n, k[:, :, :1], v[:, :, :1]), lambda: fba.cache_evict(some, table, n, 4)):
                with pytest.raises((TypeError, ValueError), match="positions"):
                    call()
