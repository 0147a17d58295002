"""rotary_func under torch's function transforms: what the autograd function refuses is refused, and a traced call is recorded, not baked in.  Gradients out of the ordinary: shared leaves, accumulated ones."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(gpu, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn((2, h, 9, 128), generator=g).to(dtype).to(gpu) for h in (4, 2)]


def test_forward_mode_is_refused(gpu):
    import flex_block_attn_amd as fba
    from torch.autograd import forward_ad

    q, k = _inputs(gpu, 0)
    turn = fba.rotary(device=gpu)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        for args in ((dual, k), (k, dual), (dual, None)):
            with pytest.raises(RuntimeError):
                fba.rotary_func(*args, turn)


def test_vmap_and_functional_gradients_are_refused(gpu):
    import flex_block_attn_amd as fba

    q, k = _inputs(gpu, 1)
    turn = fba.rotary(device=gpu)
    with pytest.raises(RuntimeError):
        torch.vmap(lambda a, b: fba.rotary_func(a, b, turn)[0])(q[None], k[None])
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda a: fba.rotary_func(a, None, turn)[0].float().sum())(q)


@pytest.mark.parametrize("shared", [False, True])
def test_traced_call_follows_its_inputs(gpu, shared):
    import flex_block_attn_amd as fba

    turn = fba.rotary((32, 64), interleaved=shared, device=gpu)
    place = lambda seed: torch.randint(-1000, 1000, (9, 2) if shared else (2, 9, 2), generator=torch.Generator().manual_seed(seed)).to(torch.int32).to(gpu)

    def f(q, k, at):
        return fba.rotary_func(q, k, turn, coordinates=at)

    traced = torch.jit.trace(f, (*_inputs(gpu, 2), place(1)), check_trace=False)
    other = (*_inputs(gpu, 3), place(2))
    for got, want in zip(traced(*other), f(*other)):
        assert torch.equal(got, want)
    got, want = (torch.jit.trace(lambda q: fba.rotary_func(q, None, turn, inverse=True)[0], (other[0],), check_trace=False)(other[0] * 2), fba.rotary_func(other[0] * 2, None, turn, inverse=True)[0])
    assert torch.equal(got, want)


class Marked(torch.Tensor):
    """A tensor subclass without semantics of its own."""


def test_tensor_subclasses_keep_their_type(gpu):
    import flex_block_attn_amd as fba

    q, k = _inputs(gpu, 4)
    turn = fba.rotary(device=gpu)
    want = fba.rotary_func(q, k, turn)
    a, b = q.as_subclass(Marked).requires_grad_(True), k.clone().requires_grad_(True)
    got = fba.rotary_func(a, b, turn)
    assert type(got[0]) is Marked and type(got[1]) is torch.Tensor
    for x, y in zip(got, want):
        assert torch.equal(x.detach().as_subclass(torch.Tensor), y)
    da, db = torch.autograd.grad(got, (a, b), [x.detach().as_subclass(torch.Tensor) for x in want])
    for x, y in zip((da, db), fba.rotary_func(*want, turn, inverse=True)):
        assert torch.equal(x.as_subclass(torch.Tensor), y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_leaf_for_both(gpu, dtype):
    """q and k of one tensor, as views of a joint projection and as the same rows twice: gradients add up."""
    import flex_block_attn_amd as fba

    g = torch.Generator().manual_seed(5)
    turn = fba.rotary((16, 56, 56), device=gpu)
    joint = torch.randn((2, 9, 6, 128), generator=g).to(dtype).to(gpu).requires_grad_(True)
    d = torch.randn((2, 9, 6, 128), generator=g).to(dtype).to(gpu)
    q, k = (x.transpose(1, 2) for x in joint.split([4, 2], 2))
    out = fba.rotary_func(q, k, turn)
    got, = torch.autograd.grad(torch.cat(out, 1).transpose(1, 2), joint, d)
    want, _ = fba.rotary_func(d.transpose(1, 2), None, turn, inverse=True)
    assert torch.equal(got, want.transpose(1, 2))
    x = joint.detach().transpose(1, 2).requires_grad_(True)
    out = fba.rotary_func(x, x, turn)
    got, = torch.autograd.grad([out[0], out[1]], x, [d.transpose(1, 2), d.transpose(1, 2)])
    assert torch.equal(got, want + want)
