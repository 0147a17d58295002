"""Attention over 4 bits with keys of all scales, those of a row far apart: values, not scales, are what is multiplied.  Against 64 bits with the bound of test_gpu_cache.py."""
import pytest
import torch

from test_gpu_cache4 import check_attend, fill, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [4, 36])
@pytest.mark.parametrize("range_of", ["small", "large"])
def test_keys_of_all_scales(gpu, dtype, heads, range_of, accumulate):
    """Up to 2^3 with a q around one, or up to the largest with a q that much smaller, so that scores have the sizes of softmax."""
    lengths = [300, 77]
    cache, table, g = make(gpu, 2, 2, 300, 16, dtype)
    fill(cache, table, lengths, g)
    limit = 13 if dtype == torch.float16 else 125
    low, high = (-limit, 3) if range_of == "small" else (-limit, limit)
    scales = torch.randint(127 + low, 127 + high + 1, cache.k_scales.shape, generator=g).to(cache.k_scales)
    cache.k_scales.copy_(torch.where(cache.k_scales != 255, scales, cache.k_scales))
    q = (torch.randn((2, heads, 1, 128), generator=g) * 2.0 ** (3 - high)).to(dtype).to(gpu)
    check_attend(q, cache, table, lengths, accumulate=accumulate)
