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


@pytest.mark.parametrize("path", range(2), ids=["native", "python"])
@pytest.mark.parametrize("H", [4, 140])  # tiles of 32 rows and keys, of 128
def test_backward_leaves_saved_tensors_as_they_are(gpu, path, H):
    leaves, do = _inputs(gpu, H, H)
    saved = []

    def keep(t):
        saved.append((t, t.detach().clone()))
        return t

    with torch.autograd.graph.saved_tensors_hooks(keep, lambda t: t):
        o = _paths()[path](*leaves)
    torch.autograd.grad(o, leaves, do)
    assert len(saved) >= 5
    for t, before in saved:
        assert torch.equal(t, before)


def test_backward_passes_of_one_forward_at_the_same_time(gpu):
    """Two captured backward passes that replay on two streams: each has statistics of its own."""
    leaves, do = _inputs(gpu, 24, 8, 1500)
    other = torch.randn(do.shape, generator=torch.Generator(device="cpu").manual_seed(9)).to(do)
    f = _paths()[0]
    want = []
    for d in (do, other):
        copies = [t.detach().clone().requires_grad_(True) for t in leaves]
        want.append(torch.autograd.grad(f(*copies), copies, d))
    torch.cuda.synchronize()
    forward, graphs, outs = torch.cuda.CUDAGraph(), [], []
    with torch.cuda.graph(forward):
        o = f(*leaves)
    for d in (do, other):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(torch.autograd.grad(o, leaves, d, retain_graph=True))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        for x in (x for out in outs for x in out):
            x.fill_(float("nan"))
        forward.replay()
        for s, graph in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            for x, y in zip(out, w):
                assert torch.equal(x, y)


def _leaf_and_way(gpu, kind):
    """(the leaves, from them to q, k and v): through a transpose each, or all from one leaf by a product, a transpose and a split."""
    g = torch.Generator(device="cpu").manual_seed(4)
    new = lambda *shape: torch.randn(shape, generator=g).to(torch.bfloat16).to(gpu)
    if kind == "transpose":
        leaves = [new(1, 100, h, 128).requires_grad_(True) for h in (4, 2, 2)]
        return leaves, lambda: [t.transpose(1, 2) for t in leaves]
    x, weight = new(1, 100, 1, 128), new(1, 100, 8, 128).requires_grad_(True)
    return [weight], lambda: (x * weight).transpose(1, 2).split((4, 2, 2), 1)


@pytest.mark.parametrize("path", range(2), ids=["native", "python"])
@pytest.mark.parametrize("kind", ["transpose", "product"])
def test_capture_beside_an_earlier_graph_of_leaves_further_away(gpu, kind, path):
    """The leaves are some steps away from the operator.  Refused while the earlier graph lives; what the pass does not come to is no reason."""
    f = _paths()[path]
    leaves, way = _leaf_and_way(gpu, kind)
    do = torch.randn((1, 4, 100, 128), generator=torch.Generator(device="cpu").manual_seed(5)).to(torch.bfloat16).to(gpu)
    earlier = f(*way())
    want = [t.clone() for t in torch.autograd.grad(earlier, leaves, do, retain_graph=True)]
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="earlier graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(f(*way()), leaves, do)
    for x, y in zip(torch.autograd.grad(earlier, leaves, do, retain_graph=True), want):
        assert torch.equal(x, y)
    # outside of a capture another stream is nobody's business
    with torch.cuda.stream(torch.cuda.Stream()):
        assert len(torch.autograd.grad(f(*way()), leaves, do)) == len(leaves)
    torch.cuda.synchronize()
    # a capture that stops at q, k and v does not come to the leaves
    parts = [t.detach() for t in way()]
    direct = torch.autograd.grad(f(*(t.requires_grad_(True) for t in parts)), parts, do)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qkv = way()
        out = torch.autograd.grad(f(*qkv), qkv, do)
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(out, direct):
        assert torch.equal(x, y)
    del earlier, qkv
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = f(*way())
        out = torch.autograd.grad(o, leaves, do)
    del o
    for _ in range(2):
        for x in out:
            x.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y)
