"""WindowAttnFunc, the Python autograd function, called by itself: it refuses what window_attn_func refuses, before a kernel gets a pointer."""
import pytest
import torch


def _apply(q, k, v, window=4, sinks=1, lengths=None):
    import flex_block_attn_amd as fba

    return fba.WindowAttnFunc.apply(q, k, v, window, sinks, True, lengths)


def test_host_tensors_are_refused():
    q = torch.zeros((1, 2, 8, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU tensor"):
        _apply(q, q, q)


@pytest.mark.gpu
def test_arguments_are_refused_as_by_the_operator(gpu):
    import flex_block_attn_amd as fba

    new = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype, device=gpu)
    q, k, n = new(1, 4, 8, 128), new(1, 2, 8, 128), torch.tensor([8], dtype=torch.int32, device=gpu)
    for error, text, args in [
        (ValueError, "GPU tensor", (q, k.cpu(), k)), (ValueError, "GPU tensor", (q.cpu(), k, k)), (TypeError, "bfloat16 or float16", (q.float(), k, k)), (ValueError, "type and device", (q, k.half(), k)),
        (ValueError, "shape", (q[0], k, k)), (ValueError, "head_dim", (new(1, 4, 8, 64), new(1, 2, 8, 64), new(1, 2, 8, 64))), (ValueError, "batch", (q, new(2, 2, 8, 128), new(2, 2, 8, 128))),
        (ValueError, "same shape", (q, k, new(1, 2, 9, 128))), (ValueError, "multiple of kv heads", (q, new(1, 3, 8, 128), new(1, 3, 8, 128))), (ValueError, "window", (q, k, k, 0)),
        (TypeError, "window", (q, k, k, 1.5)), (ValueError, "sinks", (q, k, k, 4, -1)), (ValueError, "lengths", (q, k, k, 4, 1, n.long())), (ValueError, "lengths", (q, k, k, 4, 1, n[:0])),
        (ValueError, "GPU tensor", (q, k, k, 4, 1, n.cpu())), (ValueError, "lengths", (q, new(1, 2, 9, 128), new(1, 2, 9, 128), 4, 1, n)),
    ]:
        with pytest.raises(error, match=text):
            _apply(*args)
    # as the operator: no window, and lengths that are not dense
    wide = torch.tensor([8, 3], dtype=torch.int32, device=gpu)[::2]
    assert torch.equal(_apply(q, k, k, None, 0, wide), fba.window_attn_func(q, k, k, None, lengths=wide))
