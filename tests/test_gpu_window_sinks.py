"""window_attn_func with hundreds and thousands of sinks, against the formulas in 64 bits with the bounds of test_gpu_window.py."""
import pytest
import torch

from test_gpu_window import check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B,H,Hk,Sq,Skv,window,sinks", [
    (1, 4, 2, 5000, 5000, 60, 3000),      # few tiles, many parts
    (2, 16, 16, 1500, 1500, 33, 1300),    # three parts to a tile
    (8, 32, 32, 600, 600, 40, 600),       # more tiles with sinks than work-groups: one part to a tile
    (1, 48, 24, 2100, 2100, 100, 2100),
    (8, 32, 32, 300, 600, 40, 500),
])
def test_many_sinks(gpu, causal, B, H, Hk, Sq, Skv, window, sinks):
    check(gpu, *inputs(gpu, B, H, Hk, Sq, Skv, torch.bfloat16, Sq + sinks), window, sinks, causal)


def test_many_sinks_in_padded_batches(gpu):
    lengths = torch.tensor([1500, 0, 1, 700, 1300], dtype=torch.int32, device=gpu)
    q, k, v, do = inputs(gpu, len(lengths), 24, 8, 1500, 1500, torch.float16, 6)
    check(gpu, q, k, v, do, 50, 1200, True, lengths)
