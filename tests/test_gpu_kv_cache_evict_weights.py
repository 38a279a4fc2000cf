"""GPU: rows that reach a cache without a weight, and eviction behind them."""
import pytest
import torch

import dadgpt_b200 as dad
from dadgpt_b200.attention import device_status

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("plain", [False, True], ids=["window", "plain"])
def test_a_step_without_weights_leaves_them_to_the_caller(cuda, plain):
    """Steps with weights, an eviction in place, one step without: the new row has the weight that lay there, until the caller
    sets it; the next eviction goes by what the caller has set."""
    B, H, D, budget = 3, 4, 64, 20
    g = torch.Generator(device=cuda).manual_seed(1)
    c = dad.KVCacheBF16(B, H, 64, D, device=cuda, weights=True)
    out = torch.empty(B, H, D, dtype=torch.bfloat16, device=cuda)

    def step(weights):
        x = [torch.randn(B, H, D, device=cuda, generator=g).bfloat16() for _ in range(3)]
        if plain and not weights:
            dad.decode_attention_bf16(out, *x, c, 0.125)
        else:
            dad.decode_attention_bf16_window(out, *x, c, 0.125, weights=weights)

    for _ in range(40):
        step(True)
    dad.kv_cache_evict_bf16(c, c, budget, 5)
    assert c.lengths.tolist() == [budget] * B
    left = c.weights.clone()
    step(False)
    assert torch.equal(c.weights, left)
    assert bool((left[:, :, budget] > 0).all())   # an evicted row's, or a moved one's
    c.weights[:, :, budget] = torch.tensor([0.0, 1000.0, 0.0, 1000.0], device=cuda)   # for each head
    for _ in range(8):
        step(True)
    w, k = c.weights.clone(), c.k.clone()
    dad.kv_cache_evict_bf16(c, c, budget, 5)
    n = budget + 9
    for b in range(B):
        for h in range(H):
            order = sorted(range(n - 5), key=lambda j: (-w[b, h, j].item(), j))
            stay = sorted(order[:budget - 5]) + list(range(n - 5, n))
            assert torch.equal(c.k[b, h, :budget], k[b, h, stay])
            if h % 2:
                assert budget in stay
    assert device_status() == 0


def test_behind_a_prompt_without_weights_the_first_rows_stay(cuda):
    c = dad.KVCacheBF16(2, 3, 100, 64, device=cuda, weights=True)
    c.k.normal_(generator=torch.Generator(device=cuda).manual_seed(2))
    c.lengths.fill_(80)
    k = c.k.clone()
    dad.kv_cache_evict_bf16(c, c, 30, 10)
    assert torch.equal(c.k[:, :, :20], k[:, :, :20]) and torch.equal(c.k[:, :, 20:30], k[:, :, 70:80])
