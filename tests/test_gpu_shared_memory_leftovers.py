"""GPU: results of the cache and window calls do not depend on what earlier kernels have left in shared memory."""
import pytest
import torch

import dadgpt_b200 as dad
from dadgpt_b200.attention import device_status, flash_backward_bf16_window_workspace_bytes
from tests import shared_memory
from tests.cache_reference import attend, cache_rows, check_out, visible

pytestmark = pytest.mark.gpu

LEFT = {"-inf": 0xff800000, "inf": 0x7f800000, "nan": 0x7fc00000, "3e38": 0x7f61b1e6, "-1": 0xffffffff}


def test_the_kernel_reaches_every_sm(cuda):
    assert shared_memory.fill(0).unique().numel() == torch.cuda.get_device_properties(0).multi_processor_count


# an odd number of whole blocks (half a tile at head size 64), a few first tokens, a window that ends inside a tile; one CTA
# for each (sequence, head), persistent CTAs and clusters
@pytest.mark.parametrize("left", LEFT)
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4), (64, 0), (200, 70)])
@pytest.mark.parametrize("B,H,max_len,D", [(5, 3, 400, 64), (64, 12, 400, 64), (2, 3, 2000, 64), (5, 3, 400, 128)])
def test_8_bit_decode(cuda, B, H, max_len, D, window, sinks, left):
    lengths = [[64, 192, 320, 100, 399][b % 5] for b in range(B)]
    g = torch.Generator(device=cuda).manual_seed(B)
    heads = [torch.randn(B, H, 399, D, device=cuda, generator=g).bfloat16() for _ in range(2)]
    c = dad.KVCacheFP8(B, H, max_len, D, device=cuda)
    dad.kv_cache_fill_fp8(c, *heads, torch.tensor(lengths, dtype=torch.int32, device=cuda))
    q, kn, vn = (torch.randn(B, H, D, device=cuda, generator=g).bfloat16() for _ in range(3))
    out = torch.empty_like(q)
    rows = [cache_rows(c, b, n) for b, n in enumerate(lengths)]
    torch.cuda.synchronize()
    shared_memory.fill(LEFT[left])
    dad.decode_attention_fp8(out, q, kn, vn, c, D ** -0.5, window=window, sinks=sinks)
    for b, n in enumerate(lengths):
        k, v = (torch.cat([x, new[b].double()[:, None]], 1) for x, new in zip(rows[b], (kn, vn)))
        want, _, bound, largest = attend(q[b], k, v, visible(n, n + 1, window, sinks), D ** -0.5)
        check_out(out[b], want, bound, largest)
    assert device_status() == 0


@pytest.mark.parametrize("weights", [False, True], ids=["", "weights"])
@pytest.mark.parametrize("B,H,max_len,D", [(5, 3, 400, 64), (64, 12, 400, 128), (2, 3, 2000, 64)])
def test_windowed_decode_and_eviction(cuda, B, H, max_len, D, weights):
    lengths = torch.tensor([[1, 64, 192, 333, 399][b % 5] for b in range(B)], dtype=torch.int32, device=cuda)
    results = []
    for bits in (0, *LEFT.values()):
        g = torch.Generator(device=cuda).manual_seed(B)
        c = dad.KVCacheBF16(B, H, max_len, D, device=cuda, weights=True)
        c.k.normal_(generator=g)
        c.v.normal_(generator=g)
        c.weights.exponential_(generator=g)
        q, kn, vn = (torch.randn(B, H, D, device=cuda, generator=g).bfloat16() for _ in range(3))
        got = []
        for window, sinks in ((0, 0), (70, 4)):
            out = torch.empty_like(q)
            c.lengths.copy_(lengths)
            torch.cuda.synchronize()
            shared_memory.fill(bits)
            dad.decode_attention_bf16_window(out, q, kn, vn, c, D ** -0.5, window=window, sinks=sinks, weights=weights)
            got.append(out)
        shared_memory.fill(bits)
        dad.kv_cache_evict_bf16(c, c, 150, 20)
        results.append([*got, c.k, c.v, c.weights, c.lengths])
    assert device_status() == 0
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


@pytest.mark.parametrize("D", [64, 128])
def test_windowed_attention(cuda, D):
    BH, S, scale, window, sinks = 20, 333, D ** -0.5, 70, 3
    g = torch.Generator(device=cuda).manual_seed(D)
    q, k, v, do = (torch.randn(BH, S, D, device=cuda, generator=g).bfloat16() for _ in range(4))
    ws = torch.empty(flash_backward_bf16_window_workspace_bytes(BH, S, D), dtype=torch.uint8, device=cuda)
    results = []
    for bits in (0, *LEFT.values()):
        out, dq, dk, dv = (torch.empty_like(q) for _ in range(4))
        lse = torch.empty(BH, S, device=cuda)
        shared_memory.fill(bits)
        dad.gpu_flash_attention_forward_bf16_window(out, lse, q, k, v, BH, S, D, scale, window, sinks)
        shared_memory.fill(bits)
        dad.gpu_flash_attention_backward_bf16_window(dq, dk, dv, ws, do, out, lse, q, k, v, BH, S, D, scale, window, sinks)
        results.append([out, lse, dk, dv, dq])
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0][:4], other[:4]))
        # (dQ's sums are taken in the order of arrival)
        assert (other[4].float() - results[0][4].float()).abs().max().item() <= 2.0 ** -6 * results[0][4].float().abs().max().item()
    assert device_status() == 0
