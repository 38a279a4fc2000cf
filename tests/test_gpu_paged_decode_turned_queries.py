"""GPU: a decode step over a paged cache does not round the queries that it turns: what a rounding to bf16 leaves is a second
operand. Held against float64 by bounds that a rounding of turned queries would break."""
import pytest
import torch

import dadgpt_b200 as dad
from dadgpt_b200.attention import device_status
from tests.paged_reference import attend, check, made, rows_of, turn

pytestmark = pytest.mark.gpu


def _by_head(size, K, scale):
    """max_j scale sum_d size_d |k_jd| for every query head: how far scores move when queries do by `size`."""
    group = size.shape[1] // K.shape[0]
    return torch.stack([(size[0, h] @ K[h // group].abs().T).amax() * scale for h in range(size.shape[1])])[None]


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("rot", [64, 32])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 12, 64), (24, 2, 64), (8, 2, 128), (16, 1, 128)])
@pytest.mark.parametrize("lengths", [[0, 1, 2, 15, 16, 40], [0] * 64, [700]], ids=["few rows", "first tokens", "700 rows"])
def test_scores_of_turned_queries(cuda, lengths, Hq, Hkv, D, rot, interleaved):
    """lse by large scores: of a sequence's first token it is the score. A turned query is two bf16 parts: the second is off by half
    a step of what the first left, 2^-8 of 2^-8, and both are formed from sine and cosine to 2^-20 of |x1| + |x2| (three fp32
    roundings among them)."""
    B, scale = len(lengths), 1.0
    c, _, g = made(cuda, Hkv, D, 16, lengths, [1] * B, 99)
    c.k *= 4.0
    q, k, v = (torch.randn(B, h, D, generator=g, device=cuda).mul(4.0).to(torch.bfloat16) for h in (Hq, Hkv, Hkv))
    r = dad.RotaryPositions(rot, interleaved=interleaved, device=cuda)
    out, lse = torch.empty_like(q), torch.empty(B, Hq, device=cuda)
    dad.decode_attention_paged_bf16(out, q, k, v, c, scale, rotary=r, lse=lse)
    assert device_status() == 0
    turned, size = turn(q, torch.tensor(lengths, device=cuda), r)
    rounded = turned.bfloat16().double()
    seen = 0
    for b, n in enumerate(lengths):
        K, V = rows_of(c, c.k, b, n + 1), rows_of(c, c.v, b, n + 1)
        _, want, _, bound = attend(turned[b:b + 1], K, V, n, scale, 2.0 ** -16)
        bound = bound + 2.0 ** -20 * _by_head(size[b:b + 1], K, scale)
        check(lse[b:b + 1], want, bound, f"lse of sequence {b}")
        seen += int(((attend(rounded[b:b + 1], K, V, n, scale)[1] - want).abs() > bound).sum())
    # the bounds tell the two forms apart (but at position 0, which turns by nothing: bf16 queries stay what they are)
    assert seen * 4 >= sum(n > 0 for n in lengths) * Hq
