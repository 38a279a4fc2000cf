"""GPU: the windowed backward's gradients of rows that see few keys, against float64 and the bounds for these rows."""
import pytest
import torch

import dadgpt_b200 as dad
from dadgpt_b200.attention import device_status, flash_backward_bf16_window_workspace_bytes
from tests.window_few_keys import bounds, inputs, worst

pytestmark = pytest.mark.gpu

# the first 32 rows (four warps to 16 of them), all rows, with a gap behind the first tokens and without
SHAPES = [(20, 5, 0), (32, 100, 0), (31, 0, 0), (33, 0, 0), (56, 68, 4), (40, 31, 40), (100, 16, 4), (129, 1, 31), (200, 16, 16), (300, 28, 4),
          (300, 28, 5), (300, 500, 0), (513, 32, 0), (300, 2, 200), (777, 128, 4), (1000, 256, 4), (2000, 20, 8)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,window,sinks", SHAPES)
def test_against_float64(cuda, S, window, sinks, D):
    BH, scale = 5, D ** -0.5
    g = torch.Generator(device=cuda).manual_seed(S + window + D)
    q, k, v, do = inputs(BH, S, D, g, cuda)
    out, dq, dk, dv = (torch.full_like(q, float("nan")) for _ in range(4))
    lse = torch.empty(BH, S, device=cuda)
    ws = torch.full((flash_backward_bf16_window_workspace_bytes(BH, S, D),), 0xff, dtype=torch.uint8, device=cuda)
    dad.gpu_flash_attention_forward_bf16_window(out, lse, q, k, v, BH, S, D, scale, window, sinks)
    dad.gpu_flash_attention_backward_bf16_window(dq, dk, dv, ws, do, out, lse, q, k, v, BH, S, D, scale, window, sinks)
    for u in range(BH):
        of_q, of_k = bounds(q[u], k[u], v[u], do[u], scale, window, sinks)
        assert worst(dq[u], of_q) <= 1.0
        if of_k is not None:
            assert worst(dk[u], of_k) <= 1.0
    assert device_status() == 0
