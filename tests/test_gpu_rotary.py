"""GPU: rotary positions, forward and backward, against float64."""
from fractions import Fraction

import pytest
import torch

import dadgpt_b200 as dad
from tests.paged_reference import HALF_BF16, check_turned, turn

pytestmark = pytest.mark.gpu


def _tensor(g, cuda, dtype, layout, B, S, H, D):
    """[B,S,H,D] in one of the ways in which programs keep it."""
    if layout == "heads":
        return torch.randn(B, H, S, D, generator=g, device=cuda).to(dtype).transpose(1, 2)
    if layout == "qkv":   # a slice of what one projection wrote
        return torch.randn(B, S, H + 3, D + 16, generator=g, device=cuda).to(dtype)[:, :, 2:2 + H, 16:]
    return torch.randn(B, S, H, D, generator=g, device=cuda).to(dtype)


CASES = [(1, 1, 1, 1, 16, 16), (2, 70, 4, 4, 32, 32), (3, 33, 12, 12, 64, 64), (2, 129, 8, 2, 128, 64), (1, 1000, 5, 1, 96, 48),
         (2, 5, 3, 0, 256, 256), (1, 3, 71, 71, 64, 32), (5, 1, 2, 2, 80, 16), (16, 300, 12, 12, 64, 64), (1, 2000, 32, 8, 128, 128)]


@pytest.mark.parametrize("layout", ["tokens", "heads", "qkv"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_forward_and_backward(cuda, case, dtype, interleaved, layout):
    B, S, H, Hk, D, rot = case
    g = torch.Generator(device=cuda).manual_seed(sum(case))
    r = dad.RotaryPositions(rot, interleaved=interleaved, scaling="parts", stretch=8.0, trained_len=500, device=cuda)
    q = _tensor(g, cuda, dtype, layout, B, S, H, D)
    k = _tensor(g, cuda, dtype, layout, B, S, Hk, D) if Hk else None
    q0 = q.clone()
    first = 7 * S
    positions = torch.arange(first, first + S, device=cuda).expand(B, S)
    given = None
    if layout == "heads":   # positions of each token instead, some of them negative
        given = torch.randint(-3000, 100000, (B, S), generator=g, device=cuda, dtype=torch.int32)
        positions = given
    for call, sign in ((dad.rotary_forward, 1), (dad.rotary_backward, -1)):
        qo = torch.full((B, S, H, D), 9.0, dtype=dtype, device=cuda)
        ko = torch.full((B, S, Hk, D), 9.0, dtype=dtype, device=cuda) if Hk else None
        call(qo, ko, q, k, r, positions=given, first=first if given is None else 0)
        for got, x in ((qo, q), (ko, k)):
            if x is not None:
                check_turned(got, *turn(x, positions, r, sign))
                assert torch.equal(got[..., rot:], x[..., rot:])   # the rest passes bit for bit
        assert torch.equal(q, q0)
    # in place
    want_q, want_k = torch.empty_like(q0), None if k is None else torch.empty_like(k)
    dad.rotary_forward(want_q, want_k, q, k, r, positions=given, first=first if given is None else 0)
    dad.rotary_forward(q, k, q, k, r, positions=given, first=first if given is None else 0)
    assert torch.equal(q, want_q) and (k is None or torch.equal(k, want_k))


def test_backward_is_the_transposed_forward(cuda):
    """The forward is linear: <dy, forward(x)> = <backward(dy), x>, and differences of the loss are its gradient."""
    g = torch.Generator(device=cuda).manual_seed(3)
    r = dad.RotaryPositions(32, interleaved=True, factor=1.3, device=cuda)
    x, dy, e = (torch.randn(2, 50, 4, 64, generator=g, device=cuda) for _ in range(3))
    y, dx, ye = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    dad.rotary_forward(y, None, x, None, r)
    dad.rotary_backward(dx, None, dy, None, r)
    dad.rotary_forward(ye, None, x + 0.5 * e, None, r)
    size = (dy.double().abs() * (y.double().abs() + 2 * x.double().abs())).sum()
    assert abs((dy.double() * y.double()).sum() - (dx.double() * x.double()).sum()) <= 2.0 ** -19 * size
    moved = (dy.double() * (ye.double() - y.double())).sum()
    assert abs(moved - 0.5 * (dx.double() * e.double()).sum()) <= 2.0 ** -18 * (size + (dy.abs() * e.abs()).double().sum() * 2)


@pytest.mark.parametrize("far", [1000003, 2 ** 30 + 12345, -(2 ** 31) + 5])
def test_far_positions(cuda, far):
    """Angles of far positions, from fractions: a turn's fraction keeps all of them."""
    r = dad.RotaryPositions(128, base=10000.0, device=cuda)
    x = torch.zeros(1, 1, 1, 128, device=cuda)
    x[..., :64] = 1.0   # y = (cos, sin)
    y = torch.empty_like(x)
    dad.rotary_forward(y, None, x, None, r, positions=torch.tensor([[far]], dtype=torch.int32, device=cuda))
    pi = Fraction(31415926535897932384626433832795028841971693993751, 10 ** 49)
    for i, w in enumerate(r.freq.tolist()):
        turns = far * Fraction(w) / (2 * pi)
        turns -= turns.numerator // turns.denominator
        angle = torch.tensor(float(turns * 2 * pi), dtype=torch.float64)
        # the fraction of a turn per position: half a unit of 2^-64, and its forming in 64 bits of mantissa, times the position
        allowed = 2.0 ** -21 + 6.3 * abs(far) * (2.0 ** -62 * w + 2.0 ** -65)
        assert abs(y[0, 0, 0, i].item() - torch.cos(angle).item()) <= allowed
        assert abs(y[0, 0, 0, 64 + i].item() - torch.sin(angle).item()) <= allowed


def test_ahead_of_attention_in_training(cuda):
    """Turned in place ahead of the fused attention and its gradients turned back behind it: the run of calls of a training
    step, against float64 autograd on the same bf16 queries and keys."""
    B, H, S, D = 2, 3, 200, 64
    g = torch.Generator(device=cuda).manual_seed(8)
    r = dad.RotaryPositions(D, device=cuda)
    q, k, v, do = (torch.randn(B * H, S, D, generator=g, device=cuda).to(torch.bfloat16) for _ in range(4))
    split = lambda x: x.view(B, H, S, D).transpose(1, 2)   # noqa: E731
    qt, kt, out, dq, dk, dv = (torch.empty_like(q) for _ in range(6))
    lse = torch.empty(B * H, S, device=cuda)
    ws = torch.empty(dad.attention.flash_backward_bf16_workspace_bytes(B * H, S, D), dtype=torch.uint8, device=cuda)
    dad.rotary_forward(split(qt), split(kt), split(q), split(k), r)
    dad.gpu_flash_attention_forward_bf16(out, lse, qt, kt, v, B * H, S, D, D ** -0.5)
    dad.gpu_flash_attention_backward_bf16(dq, dk, dv, ws, do, out, lse, qt, kt, v, B * H, S, D, D ** -0.5)
    dad.rotary_backward(split(dq), split(dk), split(dq), split(dk), r)
    x = [t.double().requires_grad_() for t in (q, k, v)]
    at = torch.arange(S, device=cuda)
    turned = [turn(split(t), at.expand(B, S), r)[0].transpose(1, 2).reshape(B * H, S, D) for t in x[:2]]
    s = (turned[0] @ turned[1].mT * D ** -0.5).masked_fill(at > at[:, None], float("-inf"))
    want = torch.softmax(s, -1) @ x[2]
    want.backward(do.double())
    # the attention's own bounds (relative L2 3e-2), roundings of the turned tensors and of the gradients included
    for got, ref in ((out, want.detach()), (dq, x[0].grad), (dk, x[1].grad), (dv, x[2].grad)):
        assert float((got.double() - ref).norm() / ref.norm()) <= 3e-2


def test_refusals(cuda):
    r = dad.RotaryPositions(32, device=cuda)
    x = torch.zeros(2, 5, 4, 64, device=cuda)
    y = torch.empty_like(x)
    with pytest.raises(ValueError, match="rows of neighbouring elements"):
        dad.rotary_forward(y, None, torch.zeros(2, 5, 4, 128, device=cuda)[..., ::2], None, r)
    with pytest.raises(ValueError, match="shape"):
        dad.rotary_forward(y[:1], None, x, None, r)
    with pytest.raises(ValueError, match="torch.float32"):
        dad.rotary_forward(y, None, x.bfloat16(), None, r)
    with pytest.raises(ValueError, match="positions"):
        dad.rotary_forward(y, None, x, None, r, positions=torch.zeros(5, dtype=torch.int32, device=cuda))
    with pytest.raises(RuntimeError, match="16 bytes"):
        dad.rotary_forward(y, None, torch.zeros(2, 5, 4, 66, device=cuda)[..., 1:65], None, r)
    with pytest.raises(RuntimeError, match="over each other"):
        dad.rotary_forward(torch.empty(2, 5, 1, 64, device=cuda).expand(2, 5, 4, 64), None, x, None, r)
    with pytest.raises(ValueError, match="turns"):
        bad = dad.RotaryPositions(32, device=cuda)
        bad.turns = bad.turns[:3]
        dad.rotary_forward(y, None, x, None, bad)
    # a broadcast input is read as it is
    one = torch.randn(2, 5, 1, 64, device=cuda)
    dad.rotary_forward(y, None, one.expand(2, 5, 4, 64), None, r)
    z = torch.empty_like(one)
    dad.rotary_forward(z, None, one, None, r)
    assert torch.equal(y, z.expand_as(y))


def test_captured_and_on_another_stream(cuda):
    r = dad.RotaryPositions(64, device=cuda)
    x = torch.randn(2, 40, 4, 64, device=cuda).to(torch.bfloat16)
    want, got = torch.empty_like(x), torch.empty_like(x)
    dad.rotary_forward(want, None, x, None, r, first=9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        dad.rotary_forward(got, None, x, None, r, first=9)
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and HALF_BF16 > 0
