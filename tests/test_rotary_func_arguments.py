"""RotaryFunc, the Python autograd function, called by itself: it refuses what rotary_func refuses, before a kernel gets a pointer."""
from dataclasses import replace

import pytest
import torch


def _apply(q, k, turn, coordinates=None, inverse=False):
    import flex_block_attn_amd as fba

    return fba.RotaryFunc.apply(q, k, turn.turns, turn.axes, turn.n_axes, turn.interleaved, coordinates, inverse)


def test_host_tensors_are_refused():
    import flex_block_attn_amd as fba

    turn, x = fba.rotary(device="cpu"), torch.zeros((1, 2, 8, 128), dtype=torch.bfloat16)
    for q, k in ((x, None), (x, x), (x[:, :0], x)):
        with pytest.raises(ValueError, match="GPU tensor"):
            _apply(q, k, turn)


def test_the_native_call_refuses_too():
    """On the host, where there is nothing that it could take: not even with no rows of q, whatever k is."""
    import flex_block_attn_amd as fba
    from flex_block_attn_amd import _lib

    turn, x = fba.rotary(device="cpu"), torch.zeros((1, 2, 8, 128), dtype=torch.bfloat16)
    for q, k in ((x, None), (x, x), (x[:, :0], x), (x[:, :0], x[:, :, :4]), (x[:, :0], None), (x.float(), None), (x[0], None)):
        with pytest.raises(ValueError, match="as they were"):
            _lib.host().rotary_forward(q, k, turn.turns, turn.axes, 1, True, None, False)


@pytest.mark.gpu
def test_arguments_are_refused_as_by_the_operator(gpu):
    import flex_block_attn_amd as fba
    from flex_block_attn_amd import _lib

    z = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype, device=gpu)
    turn = fba.rotary((16, 56, 56), device=gpu)
    x, where = z(2, 3, 5, 128), z(5, 3, dtype=torch.int32)
    for error, text, args in [
        (TypeError, "bfloat16 or float16", (x.float(), None, turn)), (ValueError, "q's type", (x, x.half(), turn)), (ValueError, "shape", (x[0], None, turn)),
        (ValueError, "shape", (x, x[:1], turn)), (ValueError, "shape", (x, x[:, :, :4], turn)), (ValueError, "shape", (x, x[..., :64], turn)), (ValueError, "shape", (x[:, :0], x[:, :, :4], turn)),
        (ValueError, "shape", (x[:, :0], x[:1], turn)), (ValueError, "GPU tensor", (x, x.cpu(), turn)), (ValueError, "GPU tensor", (x.cpu(), x, turn)), (ValueError, "GPU tensor", (x[:, :0], x.cpu(), turn)),
        (ValueError, "turns", (x, None, replace(turn, turns=turn.turns.int()))), (ValueError, "turns", (x, None, replace(turn, turns=turn.turns.cpu()))),
        (ValueError, "turns", (x[:, :0], x, replace(turn, turns=turn.turns.cpu()))), (ValueError, "axes", (x, None, replace(turn, axes=turn.axes.long()))),
        (ValueError, "one length", (x, None, replace(turn, axes=turn.axes[:8]))), (ValueError, "one length", (x[:, :0], x, replace(turn, axes=turn.axes[:8]))),
        (ValueError, "n_axes", (x, None, replace(turn, n_axes=0))), (ValueError, "n_axes", (x, None, replace(turn, n_axes=9))),
        (ValueError, "coordinates", (x, None, turn, where.long())), (ValueError, "coordinates", (x, None, turn, where[:4])), (ValueError, "coordinates", (x, None, turn, where[:, :2])),
        (ValueError, "coordinates", (x, None, turn, z(3, 5, 3, dtype=torch.int32))), (ValueError, "coordinates", (x[:, :0], x, turn, where[:4])), (ValueError, "coordinates", (x, None, turn, where.cpu())),
        (_lib.FbaError, "2\\^27", (z(1, 1, 1, 128).expand(1 << 14, 1, 1 << 14, 128), None, turn)),
    ]:
        with pytest.raises(error, match=text):
            _apply(*args)
    # as the operator: coordinates that are not dense
    x, where = torch.randn((2, 3, 5, 128), device=gpu).bfloat16(), torch.arange(30, dtype=torch.int32, device=gpu).reshape(5, 6)[:, ::2]
    for got, want in zip(_apply(x, x, turn, where), fba.rotary_func(x, x, turn, coordinates=where)):
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_unpacked_tensors_are_checked(gpu):
    """What a saved-tensor hook hands back goes through the same checks, on either path."""
    import flex_block_attn_amd as fba

    turn = fba.rotary((16, 56, 56), device=gpu)
    where = torch.zeros((2, 5, 3), dtype=torch.int32, device=gpu)
    for way in (lambda q, k: _apply(q, k, turn, where), lambda q, k: fba.rotary_func(q, k, turn, coordinates=where)):
        for change in (lambda t: t.cpu(), lambda t: t[:4] if t.dim() == 1 else t, lambda t: t if t.dim() == 1 else t[:1], lambda t: t if t.dim() == 1 else t[:, :4], lambda t: t if t.dim() == 1 else t.long(),
                       lambda t: t.to(torch.int16)):
            q, k = (torch.zeros((2, h, 5, 128), dtype=torch.bfloat16, device=gpu, requires_grad=True) for h in (3, 1))
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
                out = way(q, k)
            with pytest.raises(ValueError):
                torch.autograd.grad(out, (q, k), [torch.zeros_like(o) for o in out])
