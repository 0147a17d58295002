"""window_attn_func at the largest number of work-groups that a launch takes, and one sequence more."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_as_many_short_sequences_as_a_launch_takes(gpu):
    import flex_block_attn_amd as fba
    from flex_block_attn_amd import _lib

    most = 2**24 - 257
    rows = torch.randn((4096, 1, 1, 128), generator=torch.Generator(device="cpu").manual_seed(1)).to(torch.bfloat16).to(gpu)
    x = rows.repeat(-(-most // 4096) + 1, 1, 1, 1)[: most + 1]
    assert torch.equal(fba.window_attn_func(x[:most], x[:most], x[:most], 4, sinks=1), x[:most])  # a single key has all the weight
    with pytest.raises(_lib.FbaError, match="launch"):
        fba.window_attn_func(x, x, x, 4, sinks=1)


@pytest.mark.parametrize("grad", [False, True])
def test_lengths_beyond_32_bits_are_refused(gpu, grad):
    """A tensor that repeats one row costs nothing, however long it is; its length was cut to 32 bits."""
    import flex_block_attn_amd as fba
    from flex_block_attn_amd import _lib

    row = torch.ones((1, 1, 1, 128), dtype=torch.bfloat16, device=gpu)
    long, many = row.expand(1, 1, 2**32 + 5, 128), row.expand(1, 2**32 + 1, 1, 128)
    q = torch.ones((1, 1, 5, 128), dtype=torch.bfloat16, device=gpu).requires_grad_(grad)
    with pytest.raises(_lib.FbaError, match="2\\^28"):
        fba.window_attn_func(q, long, long, 4)
    with pytest.raises((_lib.FbaError, ValueError), match="2\\^28|multiple"):
        fba.window_attn_func(q, many, many, 4)
