"""window_attn_func inside of larger autograd programs: gradients of gradients, saved tensors, captured steps beside earlier graphs.  Both ways into the operator, the native
node and the Python one, have to answer alike, and so does what Python prepares first (rows that are not aligned)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(gpu, H=4, Hk=2, S=100, dtype=torch.bfloat16, seed=3):
    g = torch.Generator(device="cpu").manual_seed(seed)
    q, k, v, do = (torch.randn((1, h, S, 128), generator=g).to(dtype).to(gpu) for h in (H, Hk, Hk, H))
    return [t.requires_grad_(True) for t in (q, k, v)], do


def _paths():
    import flex_block_attn_amd as fba

    unaligned = lambda t: torch.nn.functional.pad(t, (1, 0))[..., 1:]
    return [lambda q, k, v: fba.window_attn_func(q, k, v, 30, sinks=3), lambda q, k, v: fba.WindowAttnFunc.apply(q, k, v, 30, 3, True, None),
            lambda q, k, v: fba.window_attn_func(*(unaligned(t) for t in (q, k, v)), 30, sinks=3)]


@pytest.mark.parametrize("path", range(3), ids=["native", "python", "prepared"])
def test_second_derivatives_are_refused(gpu, path):
    """A loss that contains a gradient raises when it is differentiated, instead of going without that term; a graph that is made and not differentiated changes nothing."""
    f = _paths()[path]
    leaves, do = _inputs(gpu)
    want = torch.autograd.grad(f(*leaves), leaves, do)
    o = f(*leaves)
    grads = torch.autograd.grad(o, leaves, do, create_graph=True)
    for x, y in zip(grads, want):
        assert torch.equal(x, y)
    for x in grads:
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(o.float().sum() + x.float().square().sum(), leaves, retain_graph=True, allow_unused=True)
    # the gradient of o is what is differentiated
    weight = do.clone().requires_grad_(True)
    dq, = torch.autograd.grad(f(*leaves), leaves[:1], weight, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(dq.float().sum(), weight)
    # leaves' own gradients can be used as always
    f(*leaves).backward(do, create_graph=True)
    for t, y in zip(leaves, want):
        assert torch.equal(t.grad, y)
        t.grad = None
