"""GPU: the calls on rotary positions and on a paged KV cache read nothing ahead of what the kernel ahead of them writes late."""
import pytest
import torch

import dadgpt_b200 as dad
from dadgpt_b200.attention import device_status
from tests import kernel_ahead
from tests.paged_reference import made

pytestmark = pytest.mark.gpu


def _late(call, result, targets):
    """call() gives the same `result` whichever of the targets is written by a kernel that ends late."""
    call()
    want = result().clone()
    for target in targets:
        source = target.clone()
        if target.dtype in (torch.int32, torch.int64):
            target.zero_()
        else:
            target.fill_(float("nan"))
        torch.cuda.synchronize()
        kernel_ahead.launch(target, source)
        call()
        assert torch.equal(result(), want)
    assert device_status() == 0


def test_rotary(cuda):
    g = torch.Generator(device=cuda).manual_seed(1)
    q = torch.randn(2, 50, 3, 64, generator=g, device=cuda).bfloat16()
    positions = torch.randint(0, 1000, (2, 50), generator=g, device=cuda, dtype=torch.int32)
    r = dad.RotaryPositions(64, device=cuda)
    out = torch.empty_like(q)
    _late(lambda: dad.rotary_forward(out, None, q, None, r, positions=positions), lambda: out, [q, positions, r.turns])


def test_append_and_advance(cuda):
    c, starts, g = made(cuda, 2, 64, 16, [20, 3], [40, 9], 2)
    k, v = (torch.randn(49, 2, 64, generator=g, device=cuda).bfloat16() for _ in range(2))
    r = dad.RotaryPositions(64, device=cuda)
    k0 = c.k.clone()
    dad.kv_cache_append_paged(c, k, v, starts, rotary=r)
    want = c.k.clone()
    for target in (k, starts, c.lengths, c.page_table, r.turns):
        source = target.clone()
        target.zero_()
        c.k.copy_(k0)
        torch.cuda.synchronize()
        kernel_ahead.launch(target, source)
        dad.kv_cache_append_paged(c, k, v, starts, rotary=r)
        assert torch.equal(c.k, want)
    for target in (starts, c.lengths):
        source, lengths = target.clone(), c.lengths.clone()
        target.zero_()
        torch.cuda.synchronize()
        kernel_ahead.launch(target, source)
        dad.kv_cache_advance_paged(c, starts, 49)
        assert c.lengths.tolist() == [60, 12]
        c.lengths.copy_(lengths)
    assert device_status() == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("counts", [[40, 9], [400, 3] * 40], ids=["few", "many"])
def test_attention(cuda, D, counts):
    ahead = [20, 3] * (len(counts) // 2)
    c, starts, g = made(cuda, 2, D, 16, ahead, counts, 3)
    q = torch.randn(sum(counts), 4, D, generator=g, device=cuda).bfloat16()
    out = torch.zeros_like(q)
    _late(lambda: dad.paged_attention_bf16(out, q, c, starts, max(counts), 0.125), lambda: out,
          [q, c.lengths, starts, c.page_table] + ([c.k, c.v] if len(counts) == 2 else []))


@pytest.mark.parametrize("ahead", [[20, 300], [5, 400, 77] * 60], ids=["few", "many"])
def test_decode(cuda, ahead):
    c, _, g = made(cuda, 2, 64, 16, ahead, [1] * len(ahead), 4)
    q, k, v = (torch.randn(len(ahead), h, 64, generator=g, device=cuda).bfloat16() for h in (8, 2, 2))
    r = dad.RotaryPositions(64, device=cuda)
    out = torch.zeros_like(q)
    _late(lambda: dad.decode_attention_paged_bf16(out, q, k, v, c, 0.125, rotary=r), lambda: out,
          [q, k, v, c.lengths, c.page_table, r.turns] + ([c.k, c.v] if len(ahead) == 2 else []))
