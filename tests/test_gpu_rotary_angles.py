"""GPU: sine and cosine of rotary positions in fp32, read off by turning unit vectors."""
import pytest
import torch

import dadgpt_b200 as dad

pytestmark = pytest.mark.gpu

# What sin_cos_eighth is off by (5.9e-8, over all its arguments), and the angle's conversion to fp32 (2^-28 turns); a product with
# 1 and one with 0 add nothing.
OFF = 5.9e-8 + 2.0 ** -28 * 6.2832


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("first", [-2000, 0, 10 ** 6])
def test_unit_vectors(cuda, first, interleaved):
    S, D = 20000, 64
    r = dad.RotaryPositions(D, interleaved=interleaved, device=cuda)
    x = torch.zeros(1, S, 1, D, device=cuda)
    one, two = (slice(0, D, 2), slice(1, D, 2)) if interleaved else (slice(0, D // 2), slice(D // 2, D))
    x[..., one] = 1.0
    y = torch.empty_like(x)
    dad.rotary_forward(y, None, x, None, r, first=first)
    angle = (first + torch.arange(S, device=cuda, dtype=torch.float64))[:, None] * r.freq.to(cuda)   # (to 2^-32 radians)
    assert float((y[0, :, 0, one].double() - torch.cos(angle)).abs().max()) <= OFF
    assert float((y[0, :, 0, two].double() - torch.sin(angle)).abs().max()) <= OFF
