"""GPU: one decode step over a paged KV cache, against float64."""
import pytest
import torch

import dadgpt_b200 as dad
from dadgpt_b200.attention import device_status
from tests.paged_reference import HALF_BF16, attend, check, check_turned, made, rows_of, turn

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")

# Hq, Hkv, D, page, lengths
CASES = [(1, 1, 64, 16, [0]), (1, 1, 128, 16, [1]), (12, 12, 64, 16, [700]), (12, 12, 64, 64, [0, 1, 15, 16, 63, 64, 65, 127, 128, 1000]),
         (8, 2, 128, 64, [5000, 17]), (32, 8, 128, 64, [300] * 8), (6, 2, 64, 32, [95, 96, 97]), (71, 1, 64, 128, [200, 127]),
         (17, 1, 128, 1024, [1023, 1024, 1500]), (5, 5, 64, 16, [333] * 200), (24, 3, 128, 32, [60, 2000, 31, 32]),
         (16, 16, 128, 128, [40] * 64), (2, 2, 64, 256, [60000])]


def _inputs(g, cuda, B, Hq, Hkv, D):
    return [torch.randn(B, h, D, generator=g, device=cuda).to(torch.bfloat16) for h in (Hq, Hkv, Hkv)]


def _check(c, out, lse, q, q_off, lengths, scale, sequences=None):
    for b in sequences if sequences is not None else range(len(lengths)):
        n = lengths[b] + 1
        o, s, ob, sb = attend(q[b:b + 1], rows_of(c, c.k, b, n), rows_of(c, c.v, b, n), lengths[b], scale, q_off)
        check(out[b:b + 1], o, ob, f"out of sequence {b}")
        if lse is not None:
            check(lse[b:b + 1], s, sb, f"lse of sequence {b}")


@pytest.mark.parametrize("garbage", [None, NAN, INF], ids=["old rows", "nan", "inf"])
@pytest.mark.parametrize("rotate", [False, True], ids=["", "turned"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:4])) + f"-{len(c[4])}")
def test_decode(cuda, case, rotate, garbage):
    Hq, Hkv, D, page, lengths = case
    B, scale = len(lengths), D ** -0.5
    c, _, g = made(cuda, Hkv, D, page, lengths, [1] * B, 11, garbage=garbage)
    q, k, v = _inputs(g, cuda, B, Hq, Hkv, D)
    r = dad.RotaryPositions(D // 2, interleaved=page > 16, device=cuda) if rotate else None
    out = torch.full_like(q, 9.0)
    lse = torch.empty(B, Hq, device=cuda)
    k0, v0 = c.k.clone(), c.v.clone()
    dad.decode_attention_paged_bf16(out, q, k, v, c, scale, rotary=r, lse=lse)
    at = torch.tensor(lengths, device=cuda)
    where = c.page_table[torch.arange(B, device=cuda), at // page].long()
    row = at % page
    qs, q_off = q.double(), 0.0
    if rotate:
        check_turned(c.k[where, :, row], *turn(k, at, r))
        qs, q_off = turn(q, at, r)[0], HALF_BF16 + 2.0 ** -20 * 2   # (|x1| + |x2| is at most twice sqrt(y1^2 + y2^2))
    else:
        assert torch.equal(c.k[where, :, row], k)
    assert torch.equal(c.v[where, :, row], v)
    k0[where, :, row], v0[where, :, row] = c.k[where, :, row], c.v[where, :, row]
    for now, old in ((c.k, k0), (c.v, v0)):
        assert torch.equal(now.view(torch.int16), old.view(torch.int16))
    _check(c, out, lse, qs, q_off, lengths, scale, None if B <= 10 else [0, 1, B // 2, B - 1])
    assert c.lengths.tolist() == lengths and device_status() == 0
    again = torch.empty_like(out)
    dad.decode_attention_paged_bf16(again, q, k, v, c, scale, rotary=r)   # the same step again: the same bits
    assert torch.equal(again, out)


@pytest.mark.parametrize("group", [1, 12])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 256])
@pytest.mark.parametrize("Hkv,lengths", [(1, [6001]), (3, [5500, 127]), (10, [3000]), (13, [128]), (7, [900, 641, 0, 1]),
                                         (2, [255, 257] * 17), (1, [700, 30] * 50)])
def test_ctas_with_an_sm_to_themselves(cuda, Hkv, lengths, page, D, group):
    """Eight consumer warps, tiles of 128 rows: clusters of 16, 8, 4, 2 and single CTAs."""
    B, scale = len(lengths), D ** -0.5
    c, _, g = made(cuda, Hkv, D, page, lengths, [1] * B, 21, garbage=NAN)
    q, k, v = _inputs(g, cuda, B, group * Hkv, Hkv, D)
    r = dad.RotaryPositions(D, device=cuda)
    out, lse = torch.full_like(q, 9.0), torch.empty(B, group * Hkv, device=cuda)
    dad.decode_attention_paged_bf16(out, q, k, v, c, scale, rotary=r, lse=lse)
    qs = turn(q, torch.tensor(lengths, device=cuda), r)[0]
    _check(c, out, lse, qs, HALF_BF16 + 2.0 ** -20 * 2, lengths, scale, None if B <= 10 else [0, 1, B // 2, B - 1])
    assert device_status() == 0
    again = torch.empty_like(out)
    dad.decode_attention_paged_bf16(again, q, k, v, c, scale, rotary=r)
    assert torch.equal(again, out)


@pytest.mark.parametrize("D", [64, 128])
def test_extreme_values(cuda, D):
    """Scores far apart, infinite keys and NaN: what the formula gives."""
    lengths = [300, 300, 300, 300]
    c, _, g = made(cuda, 2, D, 16, lengths, [1] * 4, 12)
    q, k, v = _inputs(g, cuda, 4, 4, 2, D)
    c.k[c.page_table[0, 3].long()] *= 40.0                      # a few scores of hundreds
    table = c.page_table.tolist()
    c.k[table[1][5], :, 2, 0] = -INF
    q[1, :, 0] = 1.0                                            # a score of minus infinity: no weight
    c.v[table[2][0], 0, 3, 7] = NAN                             # one column of one head
    q[3, 0] = 0.0
    q[3, 0, 0] = 1.0
    c.k[table[3][1], 0, 4, 0] = INF                             # a score of plus infinity: NaN
    out = torch.empty_like(q)
    dad.decode_attention_paged_bf16(out, q, k, v, c, 0.5)
    o, _, ob, _ = attend(q[:1].double(), rows_of(c, c.k, 0, 301), rows_of(c, c.v, 0, 301), 300, 0.5)
    check(out[:1], o, ob)
    K, V = rows_of(c, c.k, 1, 301), rows_of(c, c.v, 1, 301)
    keep = [j for j in range(301) if j != 5 * 16 + 2]
    o, _, ob, _ = attend(q[1:2].double(), K[:, keep], V[:, keep], 299, 0.5)
    check(out[1:2], o, ob)
    assert bool(out[2, :2, 7].isnan().all()) and not bool(out[2, 2:].isnan().any()) and not bool(out[2, :2, 8:].isnan().any())
    assert bool(out[3, 0].isnan().all()) and not bool(out[3, 2:].isnan().any())
    # the new row's own score of minus infinity
    k[0, 0, 0], q[0, :2, 0] = -INF, 1.0
    dad.decode_attention_paged_bf16(out, q, k, v, c, 0.5)
    o, _, ob, _ = attend(q[:1, :2].double(), rows_of(c, c.k, 0, 300)[:1], rows_of(c, c.v, 0, 300)[:1], 299, 0.5)
    check(out[:1, :2], o, ob)


def test_strided_tensors(cuda):
    Hq, Hkv, D, B = 6, 2, 64, 5
    lengths = [3, 100, 64, 0, 999]
    c, _, g = made(cuda, Hkv, D, 32, lengths, [1] * B, 13)
    fused = torch.randn(B, Hq + 2 * Hkv, D, generator=g, device=cuda).to(torch.bfloat16)
    q, k, v = fused[:, :Hq], fused[:, Hq:Hq + Hkv], fused[:, Hq + Hkv:]
    want = torch.empty(B, Hq, D, dtype=torch.bfloat16, device=cuda)
    dad.decode_attention_paged_bf16(want, q.contiguous(), k.contiguous(), v.contiguous(), c, 0.125)
    out = torch.full((Hq, B + 1, D + 8), 9.0, dtype=torch.bfloat16, device=cuda)
    dad.decode_attention_paged_bf16(out[:, 1:, 8:].transpose(0, 1), q, k, v, c, 0.125)
    assert torch.equal(out[:, 1:, 8:].transpose(0, 1), want)
    assert bool((out[:, 0] == 9.0).all()) and bool((out[:, :, :8] == 9.0).all())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", ["negative length", "full", "page ahead", "page of the new row"])
def test_a_sequence_that_does_not_fit_is_left_alone(cuda, what, D):
    lengths = [40, 90, 7]
    c, _, g = made(cuda, 2, D, 16, lengths, [1] * 3, 14, max_pages=6)
    q, k, v = _inputs(g, cuda, 3, 4, 2, D)
    if what == "negative length":
        c.lengths[1] = -5
    elif what == "full":
        c.lengths[1] = 96
    elif what == "page ahead":
        c.page_table[1, 2] = c.pages + 5
    else:
        c.page_table[1, 5] = -1
    k0 = c.k.clone()
    out = torch.full_like(q, 9.0)
    dad.decode_attention_paged_bf16(out, q, k, v, c, 0.125)
    assert device_status() == -1 and device_status() == 0
    assert bool((out[1] == 9.0).all())
    _check(c, out, None, q.double(), 0.0, [40, 0, 7], 0.125, [0, 2])
    if what != "page ahead":
        for b in (0, 2):
            k0[c.page_table[b, lengths[b] // 16].long(), :, lengths[b] % 16] = k[b]
        assert torch.equal(c.k, k0)
    dad.kv_cache_advance_paged(c)
    assert c.lengths[0] == 41 and c.lengths[2] == 8
    assert device_status() == (-1 if what in ("negative length", "full") else 0)


def test_shared_pages(cuda):
    """Sequences that agree in their first pages share them."""
    B, D, H = 3, 64, 2
    lengths = [70, 64, 100]
    c, _, g = made(cuda, H, D, 16, lengths, [1] * B, 15)
    c.page_table[1, :3] = c.page_table[0, :3]
    c.page_table[2, :3] = c.page_table[0, :3]
    q, k, v = _inputs(g, cuda, B, H, H, D)
    out = torch.empty_like(q)
    dad.decode_attention_paged_bf16(out, q, k, v, c, 0.125)
    _check(c, out, None, q.double(), 0.0, lengths, 0.125)


def test_two_streams_and_two_graphs(cuda):
    """Steps of two caches at once, on streams of their own and from graphs: nothing is shared between calls."""
    D, H = 64, 12
    made_ = [made(cuda, H, D, 64, [500 + 13 * i for i in range(16)], [1] * 16, 20 + i) for i in range(2)]
    ins = [_inputs(m[2], cuda, 16, H, H, D) for m in made_]
    want = [torch.empty(16, H, D, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    got = [torch.empty_like(want[0]) for _ in range(2)]
    for i in range(2):
        dad.decode_attention_paged_bf16(want[i], *ins[i], made_[i][0], 0.125)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i in range(2):
        with torch.cuda.graph(graphs[i], stream=streams[i]):
            for _ in range(5):
                dad.decode_attention_paged_bf16(got[i], *ins[i], made_[i][0], 0.125)
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].zero_()
                graphs[i].replay()
                dad.decode_attention_paged_bf16(got[i], *ins[i], made_[i][0], 0.125)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(got[i], want[i])
    assert device_status() == 0
