"""CPU: the float64 gradients that the windowed kernels are held to, against differences."""
import pytest
import torch

from tests.window_reference import backward, forward, visible


@pytest.mark.parametrize("S,window,sinks", [(1, 1, 0), (9, 3, 2), (12, 1, 0), (12, 0, 0), (10, 4, 20), (13, 5, 5)])
def test_gradients_against_differences(S, window, sinks):
    g = torch.Generator().manual_seed(S)
    q, k, v, do = (torch.randn(S, 4, generator=g, dtype=torch.float64) for _ in range(4))
    grads = backward(q, k, v, do, 0.5, window, sinks)
    loss = lambda: (forward(q, k, v, 0.5, window, sinks)[0] * do).sum().item()  # noqa: E731
    for x, grad in zip((q, k, v), grads):
        for at in range(x.numel()):
            flat = x.view(-1)
            keep = flat[at].item()
            flat[at] = keep + 1e-5
            up = loss()
            flat[at] = keep - 1e-5
            down = loss()
            flat[at] = keep
            assert abs((up - down) / 2e-5 - grad.reshape(-1)[at].item()) < 1e-8


def test_who_sees_what():
    seen = visible(6, 2, 1)
    assert seen.int().tolist() == [[1, 0, 0, 0, 0, 0], [1, 1, 0, 0, 0, 0], [1, 1, 1, 0, 0, 0], [1, 0, 1, 1, 0, 0],
                                   [1, 0, 0, 1, 1, 0], [1, 0, 0, 0, 1, 1]]
    assert torch.equal(visible(6, 0, 0), visible(6, 6, 0)) and torch.equal(visible(6, 1, 6), visible(6, 0, 0))
