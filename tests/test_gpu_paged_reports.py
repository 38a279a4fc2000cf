"""GPU: every call on a paged cache with packed batches reports a sequence whose numbers do not fit, its own rows or not."""
import pytest
import torch

import dadgpt_b200 as dad
from dadgpt_b200.attention import device_status
from tests.paged_reference import made

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("call", ["append", "attention", "advance"])
@pytest.mark.parametrize("B", [3, 300])
@pytest.mark.parametrize("what", ["negative length", "more rows than it has pages", "falling starts"])
def test_a_sequence_without_new_rows(cuda, what, B, call):
    ahead, counts = [20 + b % 5 for b in range(B)], [1 + b % 4 for b in range(B)]
    bad = B - 2
    counts[bad] = 0
    c, starts, g = made(cuda, 2, 64, 16, ahead, counts, 90)
    T = sum(counts)
    if what == "negative length":
        c.lengths[bad] = -1
    elif what == "falling starts":   # (nobody's rows: sequence bad ends ahead of its beginning, and the one behind begins there)
        starts[bad + 1] -= counts[bad - 1]
    else:
        c.lengths[bad] = c.max_pages * 16 + 1
    k, v = (torch.randn(T, 2, 64, generator=g, device=cuda).to(torch.bfloat16) for _ in range(2))
    if call == "append":
        dad.kv_cache_append_paged(c, k, v, starts)
    elif call == "attention":
        dad.paged_attention_bf16(torch.empty_like(k), k, c, starts, T, 0.125)
    else:
        dad.kv_cache_advance_paged(c, starts, T)
    assert device_status() == -1 and device_status() == 0


def test_sequences_that_fit_report_nothing(cuda):
    ahead, counts = [0, 48, 47, 0], [0, 0, 1, 48]   # full caches and empty ones
    c, starts, g = made(cuda, 2, 64, 16, ahead, counts, 91)
    k, v = (torch.randn(49, 2, 64, generator=g, device=cuda).to(torch.bfloat16) for _ in range(2))
    assert c.max_pages == 3
    dad.kv_cache_append_paged(c, k, v, starts)
    dad.paged_attention_bf16(torch.empty_like(k), k, c, starts, 48, 0.125)
    dad.kv_cache_advance_paged(c, starts, 49)
    assert device_status() == 0 and c.lengths.tolist() == [0, 48, 48, 48]
