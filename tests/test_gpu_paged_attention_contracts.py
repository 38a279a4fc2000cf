"""GPU: attention over a paged cache where rows hold infinities and NaN, behind tables wider than any sequence, and with starts
that fall, against float64."""
import pytest
import torch

import dadgpt_b200 as dad
from dadgpt_b200.attention import device_status
from tests.paged_reference import attend, check, made, rows_of

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def _call(q, c, starts, max_new, scale=0.125):
    out, lse = torch.full_like(q, 9.0), torch.full(q.shape[:2], 9.0, device=q.device)
    dad.paged_attention_bf16(out, q, c, starts, max_new, scale, lse=lse)
    assert device_status() == 0
    return out, lse


def _row(c, pool, b, j):
    """Row j of sequence b, [H, D]."""
    return pool[int(c.page_table[b, j // c.page_size]), :, j % c.page_size]


# Heads: pairs of query tiles, single ones, clusters
@pytest.mark.parametrize("H", [80, 12, 2])
@pytest.mark.parametrize("D", [64, 128])
def test_infinite_and_nan_rows(cuda, D, H):
    """Sequence 0: a NaN key, 1: a key whose score is plus infinity, 2: a NaN in V, 3: none. 300 new tokens are query tiles of 128,
    128 and 44; the row is the 200th new one, which the first tile does not see, but for sequence 2's, which is ahead of all."""
    B, ahead, n, at = 4, 70, 300, 270
    c, starts, g = made(cuda, H, D, 16, [ahead] * B, [n] * B, 95)
    q = torch.randn(B * n, H, D, generator=g, device=cuda).to(torch.bfloat16)
    q[n:2 * n, :, 0] = q[n:2 * n, :, 0].abs() + 0.5
    want, want_lse = _call(q, c, starts, n)
    _row(c, c.k, 0, at)[:, 3] = NAN
    _row(c, c.k, 1, at)[:, 0] = INF
    _row(c, c.v, 2, 5)[:, 7] = NAN
    out, lse = _call(q, c, starts, n)
    o, s, w, wl = (x.view(B, n, *x.shape[1:]) for x in (out, lse, want, want_lse))
    seen = at - ahead                                       # the first token that sees the row
    for b in (0, 1):
        assert bool(o[b, seen:].isnan().all()) and bool(s[b, seen:].isnan().all())
        # tokens ahead of it, in other tiles than those that read its tile of 128 keys (256 .. 383): as without
        clean = torch.arange(n, device=cuda) // 128 * 128 + 127 + ahead < 256
        assert int(clean.sum()) == 128 and torch.equal(o[b, clean], w[b, clean]) and torch.equal(s[b, clean], wl[b, clean])
    assert bool(o[2, :, :, 7].isnan().all()) and torch.equal(s[2], wl[2])
    rest = [d for d in range(D) if d != 7]
    assert torch.equal(o[2][..., rest], w[2][..., rest])
    assert torch.equal(o[3], w[3]) and torch.equal(s[3], wl[3])


@pytest.mark.parametrize("H", [80, 12, 2])
@pytest.mark.parametrize("D", [64, 128])
def test_scores_of_minus_infinity(cuda, D, H):
    """Rows whose first score, whose first 128 (a whole tile) or whose scores are all minus infinity."""
    B, n = 3, 200
    ahead = [40, 150, 0]
    c, starts, g = made(cuda, H, D, 16, ahead, [n] * B, 96)
    q = torch.randn(B * n, H, D, generator=g, device=cuda).to(torch.bfloat16)
    q[:, :, 0] = 1.0
    gone = [1, 128, 1]
    for b in range(B):
        for j in range(gone[b]):
            _row(c, c.k, b, j)[:, 0] = -INF
    out, lse = _call(q, c, starts, n)
    for b in range(B):
        mine = slice(b * n, (b + 1) * n)
        rows = ahead[b] + n
        K, V = rows_of(c, c.k, b, rows)[:, gone[b]:], rows_of(c, c.v, b, rows)[:, gone[b]:]
        x, o, s = q[mine].double(), out[mine], lse[mine]
        if b == 2:   # its first token sees nothing but that row
            assert bool(o[0].isnan().all()) and bool((s[0] == -INF).all())
            x, o, s = x[1:], o[1:], s[1:]
        eo, es, ob, sb = attend(x, K, V, max(ahead[b] - gone[b], 0), 0.125)
        check(o, eo, ob, f"out of sequence {b}")
        check(s, es, sb, f"lse of sequence {b}")


# Few tiles, where the calls are shared out by the most rows that there can be: Hq, Hkv, D, rows ahead, new rows
@pytest.mark.parametrize("max_pages", [None, 512, 8192], ids=["tight", "8192 rows", "131072 rows"])
@pytest.mark.parametrize("case", [(12, 12, 64, [500] * 4, [301, 1, 200, 298]), (32, 8, 128, [2256, 100, 0], [100, 21, 200]),
                                  (12, 12, 128, [0], [700]), (8, 2, 64, [33], [3]), (44, 11, 128, [600, 0], [727, 1])],
                         ids=lambda c: "x".join(map(str, c[:3])))
def test_tables_wider_than_any_sequence(cuda, case, max_pages):
    Hq, Hkv, D, ahead, counts = case
    B, T = len(counts), sum(counts)
    c, starts, g = made(cuda, Hkv, D, 16, ahead, counts, 97, max_pages=max_pages, garbage=NAN)
    q = torch.randn(T, Hq, D, generator=g, device=cuda).to(torch.bfloat16)
    out, lse = _call(q, c, starts, max(counts))
    at = 0
    for b in range(B):
        mine = slice(at, at + counts[b])
        rows = ahead[b] + counts[b]
        o, s, ob, sb = attend(q[mine].double(), rows_of(c, c.k, b, rows), rows_of(c, c.v, b, rows), ahead[b], 0.125)
        check(out[mine], o, ob, f"out of sequence {b}")
        check(lse[mine], s, sb, f"lse of sequence {b}")
        at += counts[b]
    # and a decode step behind it
    step = [torch.randn(B, h, D, generator=g, device=cuda).to(torch.bfloat16) for h in (Hq, Hkv, Hkv)]
    c.lengths += torch.tensor([n - 1 for n in counts], dtype=torch.int32, device=cuda)   # (its last row is overwritten)
    out, lse = torch.empty_like(step[0]), torch.empty(B, Hq, device=cuda)
    dad.decode_attention_paged_bf16(out, *step, c, 0.125, lse=lse)
    assert device_status() == 0
    for b in range(B):
        rows = ahead[b] + counts[b]
        o, s, ob, sb = attend(step[0][b:b + 1].double(), rows_of(c, c.k, b, rows), rows_of(c, c.v, b, rows), rows - 1, 0.125)
        check(out[b:b + 1], o, ob, f"decode, out of sequence {b}")
        check(lse[b:b + 1], s, sb, f"decode, lse of sequence {b}")


@pytest.mark.parametrize("H", [40, 2])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_that_only_one_sequence_claims_when_starts_fall(cuda, D, H):
    ahead, counts = [40, 300, 7], [200, 150, 20]
    c, starts, g = made(cuda, H, D, 16, ahead, counts, 98, max_pages=30)
    q = torch.randn(370, H, D, generator=g, device=cuda).to(torch.bfloat16)
    starts[2] = 199   # sequence 1 would end ahead of its beginning; row 199 is sequence 0's and sequence 2's
    out = torch.full_like(q, 9.0)
    dad.paged_attention_bf16(out, q, c, starts, 200, 0.125)
    assert device_status() == -1 and device_status() == 0
    o, _, ob, _ = attend(q[:200].double(), rows_of(c, c.k, 0, 240), rows_of(c, c.v, 0, 240), 40, 0.125)
    check(out[:199], o[:199], ob[:199])
