"""GPU: the 8-bit KV cache, filled by prompts and by tokens, and decode on it, against float64."""
import pytest
import torch

import dadgpt_b200 as dad
from dadgpt_b200.attention import device_status
from tests import kernel_ahead
from tests.cache_reference import BLOCK, attend, cache_rows, check_out, quantise, visible

pytestmark = pytest.mark.gpu


def _bytes(t):
    return t.contiguous().view(torch.uint8)


def _same(a, b, lengths):
    """Whether two caches hold the same rows, bit for bit."""
    for s, n in enumerate(lengths):
        w = n // BLOCK
        for x in ("k", "v"):
            assert torch.equal(_bytes(getattr(a, x))[s, :, :w * BLOCK], _bytes(getattr(b, x))[s, :, :w * BLOCK])
            assert torch.equal(getattr(a, x + "_scale")[s, :, :w], getattr(b, x + "_scale")[s, :, :w])
            assert torch.equal(getattr(a, x + "_tail")[s, :, :n % BLOCK].view(torch.int16),
                               getattr(b, x + "_tail")[s, :, :n % BLOCK].view(torch.int16))
    assert a.lengths.tolist() == b.lengths.tolist() == list(lengths)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,max_len,counts", [(1, 1, None), (63, 63, [0, 63, 5]), (64, 64, [64, 1, 0]), (200, 130, [130, 128, 129]),
                                              (301, 1000, [301, 64, 192]), (130, 130, None)])
def test_fill_against_the_format(cuda, S, max_len, counts, D, dtype):
    B, H = 3, 5
    g = torch.Generator(device=cuda).manual_seed(S)
    c = dad.KVCacheFP8(B, H, max_len, D, device=cuda)
    for t in (c.k, c.v, c.k_tail, c.v_tail):
        _bytes(t)   # (contiguous)
        t.view(torch.uint8).fill_(0x5a)
    c.k_scale.fill_(3.0)
    c.v_scale.fill_(3.0)
    heads = [torch.randn(B, H, S, D, device=cuda, generator=g) * torch.randn(B, H, S, 1, device=cuda, generator=g).exp() for _ in range(2)]
    heads = [x.to(dtype) for x in heads]
    n = [S] * B if counts is None else counts
    for b, m in enumerate(n):   # padding is not read
        for x in heads:
            x[b, :, m:] = float("nan")
    dad.kv_cache_fill_fp8(c, *heads, None if counts is None else torch.tensor(counts, dtype=torch.int32, device=cuda))
    assert c.lengths.tolist() == n and device_status() == 0
    for side, x in zip("kv", heads):
        data, scale, tail = _bytes(getattr(c, side)), getattr(c, side + "_scale"), getattr(c, side + "_tail")
        x = x.bfloat16()
        for b, m in enumerate(n):
            w = m // BLOCK
            codes, s = quantise(x[b, :, :w * BLOCK].unflatten(1, (w, BLOCK)))
            assert torch.equal(data[b, :, :w * BLOCK].cpu().unflatten(1, (w, BLOCK)), codes)
            assert torch.equal(scale[b, :, :w].cpu().double(), s)
            assert torch.equal(tail[b, :, :m - w * BLOCK], x[b, :, w * BLOCK:m])
            # what lies behind is as it was
            assert bool((data[b, :, w * BLOCK:] == 0x5a).all()) and bool((scale[b, :, w:] == 3.0).all())
            assert bool((_bytes(tail[b, :, m - w * BLOCK:]) == 0x5a).all())


def test_scales_and_codes_of_unusual_blocks(cuda):
    H, D = 9, 64
    x = torch.randn(1, H, BLOCK, D, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1))
    x[0, 0] = 0.0
    x[0, 1, 3, 4] = float("inf")
    x[0, 2, 3, 4] = float("nan")
    x[0, 3] = float("-inf")
    x[0, 4] *= 1e-38                       # denormal bf16 among them: the least scale
    x[0, 5] *= 2.0 ** 118                  # near the largest numbers
    x[0, 6] = x[0, 6].clamp(-1, 1)
    x[0, 6, 0, 0] = 1.75                   # 448 / 2^8 exactly
    x[0, 7] = x[0, 7].clamp(-1, 1)
    x[0, 7, 0, 0] = 1.7578125              # the next bf16 number
    x[0, 8] = 2.0 ** -20
    x[0, 8, 0, 0] = 448.0                  # the others round to 0
    x = x.bfloat16()
    c = dad.KVCacheFP8(1, H, 64, D, device=cuda)
    dad.kv_cache_fill_fp8(c, x, -x)
    codes, scale = quantise(x[0])
    assert torch.equal(c.k_scale[0, :, 0].cpu().double(), scale) and torch.equal(c.v_scale, c.k_scale)
    nan = torch.isnan(x[0]).cpu() | torch.isinf(x[0]).cpu()
    got = _bytes(c.k)[0].cpu()
    assert torch.equal(got[~nan], codes[~nan]) and bool(((got[nan] & 0x7f) == 0x7f).all())
    assert scale[6] * 2 == scale[7]
    got = _bytes(c.v)[0].cpu()
    assert torch.equal(got[~nan] ^ 0x80, codes[~nan]) and bool(((got[nan] & 0x7f) == 0x7f).all())


def _filled(cuda, B, H, max_len, D, lengths, seed):
    g = torch.Generator(device=cuda).manual_seed(seed)
    c = dad.KVCacheFP8(B, H, max_len, D, device=cuda)
    S = max(max(lengths), 1)
    heads = [torch.randn(B, H, S, D, device=cuda, generator=g).bfloat16() for _ in range(2)]
    dad.kv_cache_fill_fp8(c, *heads, torch.tensor(lengths, dtype=torch.int32, device=cuda))
    return c, g


def _poison(c, lengths, window, sinks):
    """Codes and scales that are NaN, and tail rows, wherever the token does not look."""
    for b, n in enumerate(lengths):
        seen = visible(n, c.max_len, window, sinks).to(c.k.device)
        whole = n // BLOCK * BLOCK
        rows = torch.arange(c.max_len, device=c.k.device)
        for data, scale, tail in ((c.k, c.k_scale, c.k_tail), (c.v, c.v_scale, c.v_tail)):
            data.view(torch.uint8)[b][:, ~seen | (rows >= whole)] = 0x7f
            used = (seen & (rows < whole)).nonzero().flatten() // BLOCK
            unused = torch.ones(scale.shape[2], dtype=torch.bool, device=c.k.device)
            unused[used] = False
            scale[b][:, unused] = float("nan")
            late = torch.ones(BLOCK, dtype=torch.bool, device=c.k.device)
            late[(seen & (rows >= whole) & (rows < n)).nonzero().flatten() % BLOCK] = False
            tail[b][:, late] = float("nan")


def _step(c, g, lengths, window, sinks, scale=None):
    B, H, D = c.B, c.H, c.D
    scale = D ** -0.5 if scale is None else scale
    q, kn, vn = (torch.randn(B, H, D, device=c.k.device, generator=g).bfloat16() for _ in range(3))
    rows = [cache_rows(c, b, n) for b, n in enumerate(lengths)]
    out = torch.full_like(q, 7.0)
    dad.decode_attention_fp8(out, q, kn, vn, c, scale, window=window, sinks=sinks)
    for b, n in enumerate(lengths):
        k, v = (torch.cat([x, new[b].double()[:, None]], 1) for x, new in zip(rows[b], (kn, vn)))
        want, _, bound, largest = attend(q[b], k, v, visible(n, n + 1, window, sinks), scale)
        check_out(out[b], want, bound, largest)
    assert c.lengths.tolist() == [n + 1 for n in lengths]
    return [n + 1 for n in lengths]


SHAPES = [(1, 3, 9000, 64, [8200]), (1, 2, 17000, 128, [16001]), (2, 5, 4100, 128, [4098, 17]),
          (8, 12, 700, 128, [0, 1, 63, 64, 65, 333, 127, 698]), (6, 7, 300, 64, [0, 63, 64, 128, 191, 255]),
          (3, 4, 40, 64, [0, 38, 5]), (64, 12, 300, 64, None), (50, 20, 90, 128, None), (300, 3, 70, 64, None)]


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (17, 4), (64, 64), (100, 70), (129, 1), (5000, 3)])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:4])))
def test_steps_against_float64(cuda, shape, window, sinks):
    B, H, max_len, D, lengths = shape
    if lengths is None:
        lengths = [(37 * b) % (max_len - 2) for b in range(B)]
    c, g = _filled(cuda, B, H, max_len, D, lengths, window + B)
    if window:
        _poison(c, lengths, window, sinks)
        _step(c, g, lengths, window, sinks)
    else:
        for _ in range(2):
            lengths = _step(c, g, lengths, window, sinks)
    assert device_status() == 0


# two sequences to a cluster of eight and of four, with one in the middle and without
@pytest.mark.parametrize("shape", [(4, 24, 1300, 64, [1298, 0, 63, 900]), (4, 24, 1300, 64, [511] * 4), (5, 20, 1300, 128, [3, 1297, 639, 0, 1250]),
                                   (9, 20, 600, 64, [0, 597, 1, 300, 319, 300, 64, 63, 575])], ids=["halves", "alike", "odd", "fours"])
def test_two_sequences_of_a_cluster(cuda, shape):
    B, H, max_len, D, lengths = shape
    c, g = _filled(cuda, B, H, max_len, D, lengths, B)
    _step(c, g, _step(c, g, lengths, 0, 0), 0, 0)
    lengths = [10 + 50 * b for b in range(B)]
    c, g = _filled(cuda, B, H, max_len, D, lengths, B + 1)
    c.lengths[0], c.lengths[B - 2] = -1, max_len
    lengths[0], lengths[B - 2] = -1, max_len
    q, kn, vn = (torch.randn(B, H, D, device=cuda, generator=g).bfloat16() for _ in range(3))
    out, before = torch.full_like(q, 7.0), c.k_tail.clone()
    dad.decode_attention_fp8(out, q, kn, vn, c, D ** -0.5)
    assert device_status() == -1
    for b, n in enumerate(lengths):
        bad = b in (0, B - 2)
        assert bool((out[b] == 7.0).all()) == bad and c.lengths[b].item() == n + (not bad)
        if not bad:
            before[b, :, n % BLOCK] = kn[b]
    assert torch.equal(c.k_tail.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("B,H,D", [(2, 3, 64), (2, 3, 128), (40, 16, 64), (160, 4, 128)])
def test_tokens_and_prompts_leave_the_same_bytes(cuda, B, H, D):
    # prompts of every length modulo a block, then as many single tokens as reach two blocks more
    max_len, steps = 260, 70
    g = torch.Generator(device=cuda).manual_seed(B)
    heads = [torch.randn(B, H, max_len, D, device=cuda, generator=g).bfloat16() for _ in range(2)]
    start = [(b * 29) % (max_len - steps) for b in range(B)]
    a, b = (dad.KVCacheFP8(B, H, max_len, D, device=cuda) for _ in range(2))
    dad.kv_cache_fill_fp8(a, *heads, torch.tensor(start, dtype=torch.int32, device=cuda))
    at = torch.tensor(start, device=cuda)
    each = torch.arange(B, device=cuda)
    out = torch.empty(B, H, D, dtype=torch.bfloat16, device=cuda)
    for s in range(steps):
        k, v = (x[each, :, at + s] for x in heads)
        dad.decode_attention_fp8(out, k, k, v, a, 0.125, window=20)
    end = [n + steps for n in start]
    dad.kv_cache_fill_fp8(b, *heads, torch.tensor(end, dtype=torch.int32, device=cuda))
    _same(a, b, end)
    assert device_status() == 0


def test_one_sequence_of_a_larger_cache(cuda):
    B, H, D, max_len = 4, 3, 64, 200
    c, g = _filled(cuda, B, H, max_len, D, [10, 100, 64, 199], 4)
    other = [t.clone() for t in (c.k.view(torch.uint8), c.k_scale, c.k_tail)]
    part = object.__new__(dad.KVCacheFP8)
    part.B, part.H, part.max_len, part.D, part.workspace = 1, H, max_len, D, c.workspace
    for x in ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail", "lengths"):
        setattr(part, x, getattr(c, x)[2:3])
    heads = [torch.randn(1, H, 150, D, device=cuda, generator=g) for _ in range(2)]
    dad.kv_cache_fill_fp8(part, *heads)
    assert c.lengths.tolist() == [10, 100, 150, 199]
    keep = [0, 1, 3]
    for now, before in zip((c.k.view(torch.uint8), c.k_scale, c.k_tail), other):
        assert torch.equal(now[keep].view(torch.uint8), before[keep].view(torch.uint8))
    _step(c, g, [10, 100, 150, 199], 0, 0)


def test_bad_counts_and_lengths_are_left_alone(cuda):
    B, H, D, max_len = 5, 2, 64, 100
    c, g = _filled(cuda, B, H, max_len, D, [7, 7, 7, 7, 7], 5)
    before = _bytes(c.k_tail).clone()
    heads = [torch.randn(B, H, 120, D, device=cuda, generator=g).bfloat16() for _ in range(2)]
    dad.kv_cache_fill_fp8(c, *heads, torch.tensor([3, -1, 101, 121, 100], dtype=torch.int32, device=cuda))
    assert device_status() == -1
    assert c.lengths.tolist() == [3, 7, 7, 7, 100] and torch.equal(_bytes(c.k_tail)[1:4], before[1:4])
    out = torch.full((B, H, D), 7.0, device=cuda).bfloat16()
    x = torch.randn(B, H, D, device=cuda, generator=g).bfloat16()
    dad.decode_attention_fp8(out, x, x, x, c, 0.125)
    assert device_status() == -1
    assert c.lengths.tolist() == [4, 8, 8, 8, 100] and bool((out[4] == 7.0).all()) and not bool((out[0] == 7.0).any())


def test_captured_and_replayed_over_a_block_s_end(cuda):
    lengths = [60, 63, 0, 126]
    c, g = _filled(cuda, 4, 12, 260, 64, lengths, 8)
    want, _ = _filled(cuda, 4, 12, 260, 64, lengths, 8)
    q, kn, vn = (torch.randn(4, 12, 64, device=cuda, generator=g).bfloat16() for _ in range(3))
    out, ref = torch.empty_like(q), torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            dad.decode_attention_fp8(out, q, kn, vn, c, 0.125)
        for step in range(6):
            graph.replay()
            dad.decode_attention_fp8(ref, q, kn, vn, want, 0.125)
            side.synchronize()
            assert torch.equal(out, ref)
            _same(c, want, [n + step + 1 for n in lengths])
    assert device_status() == 0


def test_the_kernel_ahead_may_write_everything_that_is_read(cuda):
    c, g = _filled(cuda, 2, 3, 200, 64, [150, 77], 9)
    q, kn, vn = (torch.randn(2, 3, 64, device=cuda, generator=g).bfloat16() for _ in range(3))
    out, want = torch.empty_like(q), torch.empty_like(q)
    late = c.lengths.clone()
    dad.decode_attention_fp8(want, q, kn, vn, c, 0.125)
    for target in (c.lengths, q, c.k, c.k_scale, c.v_tail):
        c.lengths.copy_(late)
        source = late if target is c.lengths else target.clone()
        target.view(torch.uint8).zero_()
        torch.cuda.synchronize()
        kernel_ahead.launch(target, source)
        dad.decode_attention_fp8(out, q, kn, vn, c, 0.125)
        assert torch.equal(out, want)
    heads = [torch.randn(2, 3, 150, 64, device=cuda, generator=g) for _ in range(2)]
    counts = torch.tensor([150, 77], dtype=torch.int32, device=cuda)
    a = dad.KVCacheFP8(2, 3, 200, 64, device=cuda)
    dad.kv_cache_fill_fp8(a, *heads, counts)
    for target in (heads[0], counts):
        source = target.clone()
        b = dad.KVCacheFP8(2, 3, 200, 64, device=cuda)
        target.zero_()
        torch.cuda.synchronize()
        kernel_ahead.launch(target, source)
        dad.kv_cache_fill_fp8(b, *heads, counts)
        _same(a, b, [150, 77])


def test_rows_behind_an_offset_of_32_bits(cuda):
    B, H, max_len, D = 2, 8200, 2200, 128
    c = dad.KVCacheFP8(B, H, max_len, D, device=cuda)
    assert c.k.numel() > 2 ** 32
    g = torch.Generator(device=cuda).manual_seed(2)
    c.k.view(torch.uint8)[1, -2:] = torch.randint(0, 127, (2, max_len, D), device=cuda, generator=g, dtype=torch.uint8)
    c.v.view(torch.uint8)[1, -2:] = torch.randint(0, 127, (2, max_len, D), device=cuda, generator=g, dtype=torch.uint8)
    c.k_scale[1, -2:] = 2.0 ** -8
    c.lengths.copy_(torch.tensor([0, 2175], dtype=torch.int32))   # the token completes the last block
    q, kn, vn = (torch.randn(B, H, D, device=cuda, generator=g).bfloat16() for _ in range(3))
    part = object.__new__(dad.KVCacheFP8)
    for x in ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail"):
        setattr(part, x, getattr(c, x)[1:, -2:].clone())
    k, v = (torch.cat([x, new[1, -2:].double()[:, None]], 1) for x, new in zip(cache_rows(part, 0, 2175), (kn, vn)))
    out = torch.empty_like(q)
    dad.decode_attention_fp8(out, q, kn, vn, c, 0.125, window=900, sinks=5)
    want, _, bound, largest = attend(q[1, -2:], k, v, visible(2175, 2176, 900, 5), 0.125)
    check_out(out[1, -2:], want, bound, largest)
    codes, scale = quantise(c.k_tail[1, -2:])
    assert torch.equal(c.k.view(torch.uint8)[1, -2:, 2112:2176].cpu(), codes)
    assert torch.equal(c.k_scale[1, -2:, 33].cpu().double(), scale)
