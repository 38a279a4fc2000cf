"""GPU: causal attention with a sliding window and first tokens that stay visible, forward and backward, against float64."""
import pytest
import torch

import dadgpt_b200 as dad
from dadgpt_b200 import _lib
from dadgpt_b200.attention import device_status, flash_backward_bf16_window_workspace_bytes, set_backward_deterministic
from tests import kernel_ahead
from tests.window_reference import backward, bounds, forward

pytestmark = pytest.mark.gpu


def _inputs(cuda, BH, S, D, seed, size=1.0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return [(torch.randn(BH, S, D, device=cuda, generator=g) * size).bfloat16() for _ in range(4)]


def _run(q, k, v, do, scale, window, sinks):
    BH, S, D = q.shape
    out, dq, dk, dv = (torch.full_like(q, float("nan")) for _ in range(4))
    lse = torch.full((BH, S), float("nan"), device=q.device)
    dad.gpu_flash_attention_forward_bf16_window(out, lse, q, k, v, BH, S, D, scale, window, sinks)
    ws = torch.full((flash_backward_bf16_window_workspace_bytes(BH, S, D),), 0xff, dtype=torch.uint8, device=q.device)
    dad.gpu_flash_attention_backward_bf16_window(dq, dk, dv, ws, do, out, lse, q, k, v, BH, S, D, scale, window, sinks)
    return out, lse, dq, dk, dv


def _check(got, inputs, scale, window, sinks, units):
    for u in units:
        one = [t[u] for t in inputs]
        out, lse, _ = forward(*one[:3], scale, window, sinks)
        want = (out, lse, *backward(*one, scale, window, sinks))
        for name, g, w, allowed in zip(("out", "lse", "dq", "dk", "dv"), got, want, bounds(*one, scale, window, sinks)):
            off = (g[u].double() - w).abs()
            assert bool((off <= allowed + 1e-30).all()), \
                f"{name} of unit {u}: off by {off.max().item()}, {(off / (allowed + 1e-30)).max().item()} of the bound"


SHAPES = [(1, 1, 0), (2, 1, 1), (63, 64, 0), (64, 17, 3), (65, 64, 1), (127, 1, 0), (128, 65, 64), (129, 128, 0), (129, 2, 130),
          (200, 63, 65), (256, 129, 4), (300, 0, 0), (300, 300, 7), (300, 5000, 0), (300, 30, 5000), (511, 128, 4),
          (500, 8, 24), (333, 32, 0), (333, 31, 2), (513, 100, 129), (640, 64, 64), (777, 256, 4), (777, 33, 300), (1000, 1, 1), (1100, 500, 0)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,window,sinks", SHAPES)
def test_against_float64(cuda, D, S, window, sinks):
    inputs = _inputs(cuda, 3, S, D, S + window)
    got = _run(*inputs, D ** -0.5, window, sinks)
    _check(got, inputs, D ** -0.5, window, sinks, range(3))
    assert device_status() == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("BH,S,window,sinks", [(200, 130, 50, 4), (96, 600, 200, 2), (7, 2500, 300, 4), (2, 9000, 1000, 70)])
def test_many_units_and_long_ones(cuda, D, BH, S, window, sinks):
    inputs = _inputs(cuda, BH, S, D, BH)
    got = _run(*inputs, D ** -0.5, window, sinks)
    _check(got, inputs, D ** -0.5, window, sinks, [0, BH // 2, BH - 1] if BH > 2 else [1])
    assert all(bool(torch.isfinite(t.float()).all()) for t in got)
    again = _run(*inputs, D ** -0.5, window, sinks)
    for name, a, b in zip(("out", "lse", "dq", "dk", "dv"), got, again):
        if name != "dq":   # (whose sums are taken in the order of arrival)
            assert torch.equal(a, b), name
    assert device_status() == 0


@pytest.mark.parametrize("D", [64, 128])
def test_large_scores(cuda, D):
    # probabilities near 1 and 0, rows whose maximum keeps growing, hidden scores far above every visible one
    inputs = _inputs(cuda, 2, 500, D, 3, size=3.0)
    inputs[1][:, :, 0] += torch.linspace(-8, 8, 500, device=cuda).bfloat16()
    inputs[0][:, :, 0] = 4.0
    inputs[1][0, 100] = 30.0
    got = _run(*inputs, D ** -0.5, 90, 3)
    _check(got, inputs, D ** -0.5, 90, 3, range(2))


@pytest.mark.parametrize("D", [64, 128])
def test_without_a_window_it_is_the_causal_call(cuda, D):
    S, scale = 333, D ** -0.5
    q, k, v, do = inputs = _inputs(cuda, 4, S, D, 5)
    got = _run(*inputs, scale, 0, 0)
    out, lse = torch.empty_like(q), torch.empty(4, S, device=cuda)
    dad.gpu_flash_attention_forward_bf16(out, lse, q, k, v, 4, S, D, scale)
    for u in range(4):
        e_out, e_lse, *_ = bounds(*(t[u] for t in inputs), scale, 0, 0)
        assert bool(((got[0][u].double() - out[u].double()).abs() <= 2 * e_out).all())
        # (the causal forward of head size 64 takes one exponential pair in eight from a cubic: 7.9e-4 of a probability)
        assert bool(((got[1][u].double() - lse[u].double()).abs() <= 2 * e_lse + 7.9e-4).all())


@pytest.mark.parametrize("D", [64, 128])
def test_what_no_query_reaches_does_not_matter(cuda, D):
    S, window, scale = 700, 64, D ** -0.5
    q, k, v, do = _inputs(cuda, 2, S, D, 6)
    want = _run(q, k, v, do, scale, window, 0)
    k2, v2, q2, do2 = (t.clone() for t in (k, v, q, do))
    for t in (k2, v2):   # the first tile of keys: queries from 128 + 128 on see none of it, nor of a tile with one of it
        t[:, :64] = float("nan")
    got = _run(q2, k2, v2, do2, scale, window, 0)
    for a, b in zip(got[:2], want[:2]):
        assert torch.equal(a[:, 256:], b[:, 256:])
    for a, b in zip(got[3:], want[3:]):   # dk, dv of keys whose queries' tiles are clean
        assert torch.equal(a[:, 512:], b[:, 512:])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,window", [(200, 1), (1, 7), (777, 1)])
def test_a_row_that_sees_one_key_has_no_gradient_of_scores(cuda, D, S, window):
    """P = 1 and dS = dP - delta = 0 for such rows. Two sums of D products in fp32, in whichever order and rounded or cut off
    (2^-23 a step), and P's own error (`rel` of bounds()) are what is left, not the rounding of out to bf16."""
    inputs = _inputs(cuda, 2, S, D, 11)
    scale = D ** -0.5
    _, lse, dq, dk, _ = _run(*inputs, scale, window, 0)
    q, k, v, do = (t.double() for t in inputs)
    size = (q * k).abs().sum(2) * scale
    rel = 2 * (D + 4) * 2.0 ** -24 * size + 2 * (S + 4) * 2.0 ** -24 + 4 * 2.0 ** -24 * lse.double().abs() + 2.0 ** -20
    ds = (2 * D * 2.0 ** -23 + 2 * rel) * (do * v).abs().sum(2) * scale * (1 + 2.0 ** -6)   # (and the roundings to bf16)
    assert bool((dq.double().abs() <= ds[..., None] * k.abs()).all()) and bool((dk.double().abs() <= ds[..., None] * q.abs()).all())


def test_a_directional_difference(cuda):
    S, D, window, sinks, scale = 150, 64, 40, 3, 0.125
    inputs = _inputs(cuda, 1, S, D, 7)
    _, _, *grads = _run(*inputs, scale, window, sinks)
    _, _, *allowed = bounds(*(t[0] for t in inputs), scale, window, sinks)
    x = [t[0].double() for t in inputs]
    g = torch.Generator(device=cuda).manual_seed(8)
    loss = lambda q, k, v: (forward(q, k, v, scale, window, sinks)[0] * x[3]).sum().item()  # noqa: E731
    for which in range(3):
        u = torch.randn(S, D, device=cuda, generator=g, dtype=torch.float64)
        up, down = [*x[:3]], [*x[:3]]
        up[which], down[which] = x[which] + 1e-5 * u, x[which] - 1e-5 * u
        slope = (loss(*up) - loss(*down)) / 2e-5
        assert abs((grads[which][0].double() * u).sum().item() - slope) <= (allowed[which] * u.abs()).sum().item() + 1e-6


def test_captured_replayed_and_on_another_stream(cuda):
    S, D, scale = 400, 64, 0.125
    inputs = _inputs(cuda, 5, S, D, 9)
    want = _run(*inputs, scale, 100, 4)
    q, k, v, do = inputs
    out, dq, dk, dv = (torch.empty_like(q) for _ in range(4))
    lse = torch.empty(5, S, device=cuda)
    ws = torch.empty(flash_backward_bf16_window_workspace_bytes(5, S, D), dtype=torch.uint8, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            dad.gpu_flash_attention_forward_bf16_window(out, lse, q, k, v, 5, S, D, scale, 100, 4)
            dad.gpu_flash_attention_backward_bf16_window(dq, dk, dv, ws, do, out, lse, q, k, v, 5, S, D, scale, 100, 4)
        for _ in range(3):
            for t in (out, lse, dq, dk, dv):
                t.fill_(float("nan"))
            graph.replay()
            side.synchronize()
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and torch.equal(dk, want[3]) and torch.equal(dv, want[4])
            assert (dq.float() - want[2].float()).abs().max().item() <= 2.0 ** -6 * want[2].float().abs().max().item()
    assert device_status() == 0


@pytest.mark.parametrize("D", [64, 128])
def test_the_kernel_ahead_may_write_everything_that_is_read(cuda, D):
    S, scale = 260, D ** -0.5
    q, k, v, do = _inputs(cuda, 2, S, D, 10)
    want = _run(q, k, v, do, scale, 70, 2)
    out, lse = torch.empty_like(q), torch.empty(2, S, device=cuda)
    for target in (q, k, v):
        source = target.clone()
        target.fill_(float("nan"))
        torch.cuda.synchronize()
        kernel_ahead.launch(target, source)
        dad.gpu_flash_attention_forward_bf16_window(out, lse, q, k, v, 2, S, D, scale, 70, 2)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    dq, dk, dv = (torch.empty_like(q) for _ in range(3))
    ws = torch.empty(flash_backward_bf16_window_workspace_bytes(2, S, D), dtype=torch.uint8, device=cuda)
    for target in (do, lse, k, ws):
        source = target.clone()
        if target is not ws:
            target.fill_(float("nan"))
        torch.cuda.synchronize()
        kernel_ahead.launch(target, source)
        dad.gpu_flash_attention_backward_bf16_window(dq, dk, dv, ws, do, out, lse, q, k, v, 2, S, D, scale, 70, 2)
        assert torch.equal(dk, want[3]) and torch.equal(dv, want[4])


def test_the_deterministic_backward_is_refused(cuda):
    S, D = 100, 64
    q, k, v, do = _inputs(cuda, 1, S, D, 11)
    out, lse = torch.empty_like(q), torch.empty(1, S, device=cuda)
    ws = torch.empty(flash_backward_bf16_window_workspace_bytes(1, S, D), dtype=torch.uint8, device=cuda)
    set_backward_deterministic(True)
    try:
        with pytest.raises(_lib.DadAttnError, match="single-pass"):
            dad.gpu_flash_attention_backward_bf16_window(q, k, v, ws, do, out, lse, q, k, v, 1, S, D, 0.125, 10, 0)
    finally:
        set_backward_deterministic(False)


def test_prompt_and_tokens_of_a_windowed_model(cuda):
    """The windowed forward over a sequence, and the same sequence as a prompt in a cache and single tokens."""
    H, S, D, prompt, window, sinks = 4, 260, 64, 150, 40, 4
    q, k, v, _ = _inputs(cuda, H, S, D, 12)
    out, lse = torch.empty_like(q), torch.empty(H, S, device=cuda)
    dad.gpu_flash_attention_forward_bf16_window(out, lse, q, k, v, H, S, D, 0.125, window, sinks)
    e_out = torch.stack([bounds(q[h], k[h], v[h], v[h], 0.125, window, sinks)[0] for h in range(H)])
    plain, small = dad.KVCacheBF16(1, H, S, D, device=cuda), dad.KVCacheFP8(1, H, S, D, device=cuda)
    plain.k[0, :, :prompt], plain.v[0, :, :prompt] = k[:, :prompt], v[:, :prompt]
    plain.lengths.fill_(prompt)
    dad.kv_cache_fill_fp8(small, k[None, :, :prompt].contiguous(), v[None, :, :prompt].contiguous())
    one, other = (torch.empty(1, H, D, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    # 8 bits: a value is off by 2^-4 of itself (or of the tiny step), a score by as much of the sum of its products' sizes
    for t in range(prompt, S):
        x, y, z = (a[None, :, t].contiguous() for a in (q, k, v))
        dad.decode_attention_bf16_window(one, x, y, z, plain, 0.125, window=window, sinks=sinks)
        dad.decode_attention_fp8(other, x, y, z, small, 0.125, window=window, sinks=sinks)
        assert bool(((one[0].double() - out[:, t].double()).abs() <= 2 * e_out[:, t]).all())
        seen = [j for j in range(t + 1) if t - j < window or j < sinks]
        ks, vs = k[:, seen].double(), v[:, seen].double()
        moved = 2.0 ** -4 * 0.125 * torch.einsum("hd,hjd->hj", q[:, t].double().abs(), ks.abs()).amax(1)
        p = torch.softmax(torch.einsum("hd,hjd->hj", q[:, t].double(), ks) * 0.125, 1)
        allowed = (torch.exp(2 * moved) - 1 + 2.0 ** -4)[:, None] * torch.einsum("hj,hjd->hd", p, vs.abs()) * 1.01 + 2 * e_out[:, t]
        assert bool(((other[0].double() - out[:, t].double()).abs() <= allowed).all())
    assert device_status() == 0
