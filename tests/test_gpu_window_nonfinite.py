"""How far a value that is infinite or no number reaches in window_attn_func: what include/fba.h states, and not beyond."""
import math

import pytest
import torch

from test_gpu_window import inputs, visible

pytestmark = pytest.mark.gpu

WINDOW, SINKS, S = 70, 4, 1100


def _step(q, k, v, do, causal):
    import flex_block_attn_amd as fba

    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o = fba.window_attn_func(*leaves, WINDOW, sinks=SINKS, causal=causal)
    return (o.detach(), *torch.autograd.grad(o, leaves, do))


def _group(index, n):  # the n rows or keys, from a multiple of n on, around each
    out = torch.zeros(S, dtype=torch.bool)
    for i in index.nonzero().flatten().tolist():
        out[i // n * n:(i // n + 1) * n] = True
    return out


def _slab_of_row(row):
    out = torch.zeros(S, dtype=torch.bool)
    out[row // 32 * 32:row // 32 * 32 + 32] = True
    if row >= S - 32:
        out[S - 32:] = True
    return out


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H", [1, 60])  # tiles of 32 rows and keys, of 128
@pytest.mark.parametrize("where", ["q", "k", "v", "do"])
@pytest.mark.parametrize("at", [2, 517, 1099])
def test_what_is_no_number_stays_near(gpu, causal, H, where, at):
    tensors = dict(zip(("q", "k", "v", "do"), inputs(gpu, 1, H, H, S, S, torch.bfloat16, 2)))
    clean = _step(**tensors, causal=causal)
    changed = dict(tensors, **{where: tensors[where].clone()})
    changed[where][0, 0, at, 5] = math.inf if at % 2 else math.nan
    got = _step(**changed, causal=causal)
    seen = visible(S, S, WINDOW, SINKS, causal)  # (rows, keys)
    here = torch.zeros(S, dtype=torch.bool)
    here[at] = True
    key_slab = _group(here, 32)
    if where in ("k", "v"):
        rows = seen[:, at]
        keys = seen[rows].any(0) | here
        reach = {"o": rows, "dq": rows, "dk": keys, "dv": keys}
        beside = _group(seen[:, key_slab].any(1), 32)
        reach["o" if where == "v" else "dq"] = beside
        if where == "v":  # rows whose o is no number have no delta
            keys = seen[beside].any(0) | here
            reach.update(dq=beside, dk=keys)
    else:
        keys = seen[at]
        reach = {"o": here if where == "q" else ~here & here, "dq": here, "dk": keys, "dv": keys}
        reach["dk" if where == "q" else "dv"] = _group(seen[_slab_of_row(at)].any(0), 128)
    for name, x, y in zip(("o", "dq", "dk", "dv"), got, clean):
        far = ~reach[name].to(gpu)
        assert torch.equal(x[0, 0, far], y[0, 0, far]), name
        assert torch.equal(x[0, 1:], y[0, 1:]), name  # other heads
    nearest = {"q": (0, 1), "k": (0, 1), "v": (0, 2), "do": (3,)}[where]  # and it does reach what sees it
    for i in nearest:
        own = seen[:, at] if where in ("k", "v") else (keys if i == 3 else here)
        assert not bool(torch.isfinite(got[i][0, 0, own.to(gpu)]).all())
