"""GPU: decode over a sliding window of a bf16 cache and with the attention weights added up, against float64."""
import pytest
import torch

import dadgpt_b200 as dad
from dadgpt_b200.attention import device_status
from tests import kernel_ahead
from tests.cache_reference import U, attend, check_out, visible

pytestmark = pytest.mark.gpu


def _cache(cuda, B, H, max_len, D, lengths, seed, weights):
    g = torch.Generator(device=cuda).manual_seed(seed)
    c = dad.KVCacheBF16(B, H, max_len, D, device=cuda, weights=weights)
    c.k.normal_(generator=g)
    c.v.normal_(generator=g)
    if weights:
        c.weights.exponential_(generator=g)
    c.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    return c, g


def _hide(c, lengths, window, sinks):
    """NaN wherever no token looks: behind the rows and between the first ones and the window."""
    for b, n in enumerate(lengths):
        hidden = ~visible(n, c.max_len, window, sinks)
        c.k[b][:, hidden.to(c.k.device)] = float("nan")
        c.v[b][:, hidden.to(c.k.device)] = float("nan")


def _step(c, g, lengths, window, sinks, weights, scale=None):
    B, H, D = c.B, c.H, c.D
    scale = D ** -0.5 if scale is None else scale
    q, kn, vn = (torch.randn(B, H, D, device=c.k.device, generator=g).bfloat16() for _ in range(3))
    out = torch.full_like(q, 7.0)
    k0, v0 = c.k.clone(), c.v.clone()
    w0 = c.weights.clone() if weights else None
    dad.decode_attention_bf16_window(out, q, kn, vn, c, scale, window=window, sinks=sinks, weights=weights)
    for b, n in enumerate(lengths):
        k0[b, :, n], v0[b, :, n] = kn[b], vn[b]
        want, p, bound, largest = attend(q[b], k0[b], v0[b], visible(n, c.max_len, window, sinks), scale)
        check_out(out[b], want, bound, largest)
        if weights:
            before = w0[b].double()
            before[:, n] = 0.0
            allowed = p * bound[:, None] + 2 * U * (before + p)
            assert bool(((c.weights[b].double() - before - p).abs() <= allowed).all())
            same = ~visible(n, c.max_len, window, sinks)
            assert torch.equal(c.weights[b][:, same.to(c.k.device)], w0[b][:, same.to(c.k.device)])
    assert torch.equal(c.k.view(torch.int16), k0.view(torch.int16)) and torch.equal(c.v.view(torch.int16), v0.view(torch.int16))
    assert c.lengths.tolist() == [n + 1 for n in lengths]
    return [n + 1 for n in lengths]


# clusters of 8, 4 and 2, one CTA each, persistent CTAs with and without ranking, more sequences than are ranked
SHAPES = [(1, 3, 9000, 64, [8200]), (2, 5, 4100, 128, [4098, 17]), (7, 12, 700, 128, [0, 1, 63, 64, 65, 333, 698]),
          (3, 4, 40, 64, [0, 38, 5]), (64, 12, 300, 64, None), (50, 20, 90, 64, None), (300, 3, 70, 128, None)]


@pytest.mark.parametrize("weights", [False, True], ids=["", "weights"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (17, 4), (64, 64), (129, 1), (5000, 3)])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:4])))
def test_steps_against_float64(cuda, shape, window, sinks, weights):
    B, H, max_len, D, lengths = shape
    if lengths is None:
        lengths = [(37 * b) % (max_len - 2) for b in range(B)]
    c, g = _cache(cuda, B, H, max_len, D, lengths, window + B, weights)
    _hide(c, lengths, window, sinks)
    lengths = _step(c, g, lengths, window, sinks, weights)
    if not window:   # (a window moves on over rows that were made NaN)
        _step(c, g, lengths, window, sinks, weights)
    assert device_status() == 0


# two sequences to a cluster of eight and of four, with one in the middle and without
PAIRED = [(4, 24, 1300, 64, [1298, 0, 17, 900]), (4, 24, 1300, 64, [500] * 4), (5, 20, 1300, 128, [3, 1297, 640, 0, 1250]),
          (9, 20, 600, 64, [0, 597, 1, 300, 300, 300, 64, 63, 590])]


@pytest.mark.parametrize("weights", [False, True], ids=["", "weights"])
@pytest.mark.parametrize("shape", PAIRED, ids=["halves", "alike", "odd", "fours"])
def test_two_sequences_of_a_cluster(cuda, shape, weights):
    B, H, max_len, D, lengths = shape
    c, g = _cache(cuda, B, H, max_len, D, lengths, B, weights)
    _hide(c, lengths, 0, 0)
    _step(c, g, _step(c, g, lengths, 0, 0, weights), 0, 0, weights)
    # no token for a full and for an invalid length, whichever of the two sequences has it
    c.k.normal_(generator=g)
    c.v.normal_(generator=g)
    for bad in ([0], [1], [B - 1], [0, 1], [2, 3], list(range(B))):
        lengths = [(1300 if i % 2 else -5) if i in bad else 10 * i for i in range(B)]
        c.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        q, kn, vn = (torch.randn(B, H, D, device=cuda, generator=g).bfloat16() for _ in range(3))
        out, k0 = torch.full_like(q, 7.0), c.k.clone()
        dad.decode_attention_bf16_window(out, q, kn, vn, c, D ** -0.5, weights=weights)
        assert device_status() == -1 and c.lengths.tolist() == [n if i in bad else n + 1 for i, n in enumerate(lengths)]
        for i, n in enumerate(lengths):
            if i in bad:
                assert bool((out[i] == 7.0).all())
            else:
                k0[i, :, n] = kn[i]
                want, _, bound, largest = attend(q[i], c.k[i], c.v[i], visible(n, max_len, 0, 0), D ** -0.5)
                check_out(out[i], want, bound, largest)
        assert torch.equal(c.k.view(torch.int16), k0.view(torch.int16))


def test_without_a_window_it_is_the_decode_call(cuda):
    lengths = [0, 5, 299, 130]
    a, g = _cache(cuda, 4, 12, 300, 64, lengths, 1, False)
    b, _ = _cache(cuda, 4, 12, 300, 64, lengths, 1, False)
    q, kn, vn = (torch.randn(4, 12, 64, device=cuda, generator=g).bfloat16() for _ in range(3))
    x, y = torch.empty_like(q), torch.empty_like(q)
    dad.decode_attention_bf16(x, q, kn, vn, a, 0.125)
    dad.decode_attention_bf16_window(y, q, kn, vn, b, 0.125)
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and torch.equal(a.lengths, b.lengths)
    assert (x.float() - y.float()).abs().max().item() <= 2.0 ** -7 * x.float().abs().max().item()


def test_the_two_calls_take_turns_on_one_workspace(cuda):
    lengths = [(11 * b) % 200 for b in range(64)]
    c, g = _cache(cuda, 64, 12, 260, 64, lengths, 3, True)
    for _ in range(3):
        q, kn, vn = (torch.randn(64, 12, 64, device=cuda, generator=g).bfloat16() for _ in range(3))
        dad.decode_attention_bf16(torch.empty_like(q), q, kn, vn, c, 0.125)
        lengths = _step(c, g, [n + 1 for n in lengths], 33, 2, True)
        lengths = _step(c, g, lengths, 0, 0, False)


@pytest.mark.parametrize("B,H,D", [(5, 3, 64), (100, 12, 128), (300, 4, 64)])
def test_full_and_invalid_sequences_are_left_alone(cuda, B, H, D):
    c, g = _cache(cuda, B, H, 33, D, [0] * B, 5, True)
    c.lengths[1], c.lengths[3] = 33, -1
    k0, w0 = c.k.clone(), c.weights.clone()
    x = torch.randn(B, H, D, device=cuda, generator=g).bfloat16()
    out = torch.full_like(x, 7.0)
    dad.decode_attention_bf16_window(out, x, x, x, c, 0.125, window=8, sinks=2, weights=True)
    assert device_status() == -1
    for b in (1, 3):
        assert bool((out[b] == 7.0).all()) and torch.equal(c.k[b], k0[b]) and torch.equal(c.weights[b], w0[b])
    keep = [i for i in range(B) if i not in (1, 3)]
    assert c.lengths.tolist() == [33 if i == 1 else -1 if i == 3 else 1 for i in range(B)]
    assert torch.equal(out[keep], x[keep]) and bool((c.weights[keep][:, :, 0] == 1.0).all())


def test_infinities_and_lowest_values_that_are_seen(cuda):
    # a row whose score is the lowest finite number, or -inf, has probability 0; an infinite value with weight shows
    c, g = _cache(cuda, 1, 2, 64, 64, [3], 6, False)
    q = torch.ones(1, 2, 64, device=cuda).bfloat16()
    c.k.zero_()
    c.k[0, 0, 1] = -1e38
    c.k[0, 0, 2] = float("-inf")
    c.v[0, 1, 0, 5] = float("inf")
    vn = torch.randn(1, 2, 64, device=cuda, generator=g).bfloat16()
    out = torch.empty_like(q)
    dad.decode_attention_bf16_window(out, q, torch.zeros_like(q), vn, c, 1.0, window=64)
    mean = (c.v[0, 0, 0].double() + vn[0, 0].double()) / 2
    assert (out[0, 0].double() - mean).abs().max().item() <= 2.0 ** -7 * mean.abs().max().item()
    assert out[0, 1, 5].item() == float("inf") and bool(torch.isfinite(out[0, 1, :5]).all())


def test_captured_on_another_stream_and_replayed(cuda):
    lengths = [200, 3, 130]
    c, g = _cache(cuda, 3, 12, 260, 64, lengths, 8, True)
    start = c.lengths.clone()
    weights = c.weights.clone()
    q, kn, vn = (torch.randn(3, 12, 64, device=cuda, generator=g).bfloat16() for _ in range(3))
    out = torch.empty_like(q)
    call = lambda: dad.decode_attention_bf16_window(out, q, kn, vn, c, 0.125, window=40, sinks=4, weights=True)  # noqa: E731
    call()
    want, w = out.clone(), c.weights.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
        for _ in range(3):
            c.lengths.copy_(start)
            c.weights.copy_(weights)
            out.zero_()
            graph.replay()
            side.synchronize()
            assert torch.equal(out, want) and torch.equal(c.weights, w) and c.lengths.tolist() == [201, 4, 131]
    assert device_status() == 0


def test_the_kernel_ahead_may_write_everything_that_is_read(cuda):
    lengths = [150, 77]
    c, g = _cache(cuda, 2, 3, 200, 64, lengths, 9, False)
    q, kn, vn = (torch.randn(2, 3, 64, device=cuda, generator=g).bfloat16() for _ in range(3))
    out, want = torch.empty_like(q), torch.empty_like(q)
    late = c.lengths.clone()
    dad.decode_attention_bf16_window(want, q, kn, vn, c, 0.125, window=50, sinks=2)
    for target, source in ((c.lengths, late), (q, q.clone()), (c.k, c.k.clone())):
        c.lengths.copy_(late)
        if target is c.lengths:
            target.zero_()
        else:
            target.fill_(float("nan"))
        torch.cuda.synchronize()
        kernel_ahead.launch(target, source)
        dad.decode_attention_bf16_window(out, q, kn, vn, c, 0.125, window=50, sinks=2)
        assert torch.equal(out, want)


def test_rows_behind_an_offset_of_32_bits(cuda):
    # 2 x 16385 heads x 1100 rows x 64: the last sequence's rows begin beyond 2^31 elements
    B, H, max_len, D = 2, 16400, 1100, 64
    c = dad.KVCacheBF16(B, H, max_len, D, device=cuda)
    assert c.k.numel() > 2 ** 31
    g = torch.Generator(device=cuda).manual_seed(2)
    c.k[1, -3:].normal_(generator=g)
    c.v[1, -3:].normal_(generator=g)
    c.lengths.copy_(torch.tensor([0, 1050], dtype=torch.int32))
    q, kn, vn = (torch.randn(B, H, D, device=cuda, generator=g).bfloat16() for _ in range(3))
    out = torch.empty_like(q)
    dad.decode_attention_bf16_window(out, q, kn, vn, c, 0.125, window=900, sinks=5)
    want, _, bound, largest = attend(q[1, -3:], c.k[1, -3:], c.v[1, -3:], visible(1050, max_len, 900, 5), 0.125)
    check_out(out[1, -3:], want, bound, largest)
    assert torch.equal(out[0], vn[0]) and torch.equal(c.k[1, :, 1050], kn[1])
