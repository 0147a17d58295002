"""Gradients of window_attn_func where softmax is saturated: scores so large that one key has all the weight of most rows.

Against the formulas in 64 bits with the bounds of test_gpu_window.py (whose e is large here, since scores are).  Beyond that, of a row whose second largest score is 40 or more
behind, in log2 units: o is the row of v that has the weight, exactly, and dS of that key is P (dP - delta) of two fp32 sums of the same 128 products, dO and v, each off by
130 * 2^-24 of their sizes at most.  P is 1 but for the rounding of a score of 2^15 at most in fp32, 2^-9 * ln 2 (and dQ is divided by the sum of P); all other keys together have less than
2^-30 of P (300 of them), with |dP - delta| at most twice the largest sum of the sizes of 128 products.  dQ is rounded once.

Weights, dS and products below 2^-126, where fp32 ends, are zeros (bf16 ends there too, so that values of that size are left in the reference): each of a sum's terms, 300 at most, is
off by 2^-126 (|dP - delta| + 2) (|factor| + 1) at most by that, with |dP - delta| as above and the factor q, k or dO.
"""
import math

import pytest
import torch

from test_gpu_window import SCALE, inputs, reference, visible

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H", [2, 140])  # tiles of 32 rows and keys, of 128
def test_gradients_of_saturated_rows(gpu, dtype, H):
    S, f = 300, 2.0**-24
    q, k, v, do = inputs(gpu, 1, H, H, S, S, dtype, 3, size=1.0)
    q = q * 1000
    import flex_block_attn_amd as fba

    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = fba.window_attn_func(*leaves, 40, sinks=3)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    o = o.detach()
    sizes = do.double().abs() @ v.double().abs().transpose(-1, -2)
    low = 2.0**-126 * 300 * (2 * float(sizes.max()) + 2)
    want, off = reference(q, k, v, do, 40, 3, True, None)
    for name, x, y, z, factor in (("o", o, want[0], off[0], v), ("dq", dq, want[1], off[1], k), ("dk", dk, want[2], off[2], q), ("dv", dv, want[3], off[3], do)):
        over = (x.double() - y).abs() - z - low * (float(factor.abs().max()) + 1)
        assert bool(torch.isfinite(x).all()) and bool((over <= 0).all()), f"{name}: {over.max().item():.3e} beyond the bound, at {(over > 0).sum().item()} of {over.numel()}"
    s = (q.double() @ k.double().transpose(-1, -2) * SCALE).masked_fill(~visible(S, S, 40, 3, True, device=gpu), -math.inf)
    assert float(s.masked_fill(s.isinf(), 0).abs().max()) * math.log2(math.e) < 2**15
    top = s.topk(2, -1)
    clear = (top.values[..., 0] - top.values[..., 1]) * math.log2(math.e) > 40
    assert int(clear.sum()) > clear.numel() // 2
    of_top = lambda t: torch.gather(t, 2, top.indices[..., :1].expand(-1, -1, -1, 128))
    ds = 260 * f * torch.gather(sizes, -1, top.indices[..., :1])
    rest = 2.0**-30 * 2 * sizes.amax(-1, keepdim=True)
    bound = 1.01 * SCALE * (ds * of_top(k).double().abs() + rest * k.double().abs().amax(2, keepdim=True)) * (1 + torch.finfo(dtype).eps) + torch.finfo(dtype).smallest_normal
    assert torch.equal(o[clear], of_top(v)[clear])
    assert bool((dq.double().abs() <= bound)[clear].all())
