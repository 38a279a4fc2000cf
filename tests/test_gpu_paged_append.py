"""GPU: new rows into a paged KV cache, turned on the way, against float64."""
import pytest
import torch

import dadgpt_b200 as dad
from dadgpt_b200.attention import device_status
from tests.paged_reference import check_turned, made, turn

pytestmark = pytest.mark.gpu

# Hq, Hkv, D, page, ahead, counts
CASES = [(4, 4, 64, 16, [0], [1]), (12, 12, 64, 16, [700], [301]), (8, 2, 128, 64, [0, 63, 64, 1000], [64, 1, 0, 130]),
         (3, 1, 64, 128, [5, 0, 0, 17, 200], [0, 0, 3, 0, 40]), (71, 71, 64, 32, [10], [2]), (2, 2, 128, 1024, [1000, 3], [100, 7]),
         (32, 8, 128, 16, list(range(300)), [i % 3 for i in range(300)]), (6, 2, 64, 64, [37, 4000], [3000, 500])]


def _places(c, ahead, counts):
    """(page, row in the page) of every new token."""
    table = c.page_table.tolist()
    page, row = [], []
    for b, (a, n) in enumerate(zip(ahead, counts)):
        page += [table[b][j // c.page_size] for j in range(a, a + n)]
        row += [j % c.page_size for j in range(a, a + n)]
    return torch.tensor(page, device=c.k.device), torch.tensor(row, device=c.k.device)


@pytest.mark.parametrize("rotate", ["no", "half", "interleaved", "part"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:4])))
def test_rows_in_their_pages(cuda, case, dtype, rotate):
    Hq, Hkv, D, page, ahead, counts = case
    c, starts, g = made(cuda, Hkv, D, page, ahead, counts, 5)
    T = sum(counts) + 2   # two rows behind the last sequence's
    q, k, v = (torch.randn(T, h, D, generator=g, device=cuda).to(dtype) for h in (Hq, Hkv, Hkv))
    r = None if rotate == "no" else dad.RotaryPositions(D // 2 if rotate == "part" else D, interleaved=rotate == "interleaved",
                                                        scaling="linear", stretch=2.0, device=cuda)
    q_out = torch.full((T, Hq, D), 9.0, dtype=torch.bfloat16, device=cuda)
    k0, v0, lengths = c.k.clone(), c.v.clone(), c.lengths.clone()
    dad.kv_cache_append_paged(c, k, v, starts, q=q, q_out=q_out, rotary=r)
    n = sum(counts)
    at = torch.tensor([j for a, m in zip(ahead, counts) for j in range(a, a + m)], device=cuda)
    where = _places(c, ahead, counts)
    if r is None:
        assert torch.equal(q_out[:n], q[:n].bfloat16()) and torch.equal(c.k[where[0], :, where[1]], k[:n].bfloat16())
    else:
        for got, x in ((q_out[:n], q[:n]), (c.k[where[0], :, where[1]], k[:n])):
            want, size = turn(x, at, r)
            check_turned(got, want, size)
    assert torch.equal(c.v[where[0], :, where[1]], v[:n].bfloat16())
    # nothing else has changed
    for now, old in ((c.k, k0), (c.v, v0)):
        old = old.clone()
        old[where[0], :, where[1]] = now[where[0], :, where[1]]
        assert torch.equal(now, old)
    assert bool((q_out[n:] == 9.0).all()) and torch.equal(c.lengths, lengths)
    dad.kv_cache_advance_paged(c, starts, T)
    assert c.lengths.tolist() == [a + m for a, m in zip(ahead, counts)] and device_status() == 0


def test_heads_of_a_prefill_and_slices_of_a_projection(cuda):
    Hq, Hkv, D, n = 6, 2, 64, 77
    c, starts, g = made(cuda, Hkv, D, 16, [20], [n], 6)
    r = dad.RotaryPositions(D, device=cuda)
    fused = torch.randn(n, Hq + 2 * Hkv, D, generator=g, device=cuda).to(torch.bfloat16)
    q, k, v = fused[:, :Hq], fused[:, Hq:Hq + Hkv], fused[:, Hq + Hkv:]
    q_out = torch.empty(n, Hq, D, dtype=torch.bfloat16, device=cuda)
    dad.kv_cache_append_paged(c, k, v, starts, q=q, q_out=q_out, rotary=r)
    want_k, want_v = c.k.clone(), c.v.clone()
    c.k.zero_(), c.v.zero_()
    heads = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]   # [H, n, D] in memory
    turned = torch.empty(Hq, n, D, dtype=torch.bfloat16, device=cuda)
    dad.kv_cache_append_paged(c, heads[1], heads[2], starts, q=heads[0], q_out=turned.transpose(0, 1), rotary=r)
    where = _places(c, [20], [n])
    for now, want in ((c.k, want_k), (c.v, want_v)):
        assert torch.equal(now[where[0], :, where[1]], want[where[0], :, where[1]])
    assert torch.equal(turned.transpose(0, 1), q_out)
    # in place, and without queries
    dad.kv_cache_append_paged(c, k, v, starts, q=q, q_out=q, rotary=r)
    assert torch.equal(q, q_out)
    c.k.zero_()
    dad.kv_cache_append_paged(c, k, v, starts, rotary=r)
    assert torch.equal(c.k[where[0], :, where[1]], want_k[where[0], :, where[1]])


@pytest.mark.parametrize("what", ["negative length", "no room", "page", "falling starts", "starts behind T", "negative page"])
def test_a_sequence_that_does_not_fit_is_left_alone(cuda, what):
    D, page, counts = 64, 16, [5, 20, 3]
    ahead = [10, 12, 40]
    c, starts, g = made(cuda, 2, D, page, ahead, counts, 7)
    assert c.max_pages == 3
    good = {0, 2}
    if what == "negative length":
        c.lengths[1] = -1
    elif what == "no room":
        c.lengths[1] = 48 - 19
    elif what == "page":
        c.page_table[1, 1] = c.pages   # rows 16 .. 31 of its rows: the others are written
    elif what == "negative page":
        c.page_table[1, 1] = -1
    elif what == "falling starts":
        starts[2] = 4                  # row 4 is sequence 0's and sequence 2's: whose it is taken for is not said
        good = {0}
    else:
        starts[3] = 100
        good = {0, 1}
    T = sum(counts)
    k, v = (torch.randn(T, 2, D, generator=g, device=cuda).to(torch.bfloat16) for _ in range(2))
    k0 = c.k.clone()
    before = c.lengths.clone()
    dad.kv_cache_append_paged(c, k, v, starts)
    assert device_status() == -1 and device_status() == 0
    changed = torch.nonzero((c.k != k0).any(-1).any(1)).tolist()   # (page, row)
    table = c.page_table.tolist()
    allowed, needed = set(), set()
    at = [0, 5, 25, 28]
    for b in range(3):
        rows = {(table[b][j // page], j % page) for j in range(ahead[b], ahead[b] + counts[b])}
        if b in good:
            needed |= rows
        allowed |= rows
    got = {tuple(x) for x in changed}
    if what in ("page", "negative page"):
        needed |= {(table[1][0], j) for j in range(12, 16)}
        assert got == needed
    elif what == "falling starts":
        assert needed - {(table[0][0], 14)} <= got
        assert c.k[table[0][0], 0, 10:14].equal(k[:4, 0])
    else:
        assert got == needed
    dad.kv_cache_advance_paged(c, starts, T)
    if what in ("negative length", "no room"):
        assert device_status() == -1 and c.lengths[1] == before[1] and c.lengths[0] == 15 and c.lengths[2] == 43
    else:
        device_status()
    assert at[-1] == T


def test_one_token_each(cuda):
    B, H, D = 40, 3, 128
    ahead = [(17 * b) % 50 for b in range(B)]
    c, _, g = made(cuda, H, D, 16, ahead, [1] * B, 9)
    k, v = (torch.randn(B, H, D, generator=g, device=cuda) for _ in range(2))
    dad.kv_cache_append_paged(c, k, v)
    where = _places(c, ahead, [1] * B)
    assert torch.equal(c.k[where[0], :, where[1]], k.bfloat16()) and torch.equal(c.v[where[0], :, where[1]], v.bfloat16())
    dad.kv_cache_advance_paged(c)
    assert c.lengths.tolist() == [a + 1 for a in ahead] and device_status() == 0
    with pytest.raises(RuntimeError, match="without starts"):
        dad.kv_cache_append_paged(c, k[:5], v[:5])
    with pytest.raises(ValueError, match="starts"):
        dad.kv_cache_append_paged(c, k, v, torch.zeros(3, dtype=torch.int32, device=cuda))
    with pytest.raises(ValueError, match="v_new"):
        dad.kv_cache_append_paged(c, k, v.bfloat16())
    with pytest.raises(ValueError, match="q_out"):
        dad.kv_cache_append_paged(c, k, v, q=k, q_out=k)


@pytest.mark.parametrize("rotate", [False, True])
def test_rows_ahead_of_the_first_sequence_belong_to_nobody(cuda, rotate):
    """starts[0] above 0: the packed rows ahead of it are another batch's, as those behind the last are."""
    Hq, Hkv, D, ahead, counts, lead = 4, 2, 64, [3, 40], [17, 1], 37
    c, starts, g = made(cuda, Hkv, D, 16, ahead, counts, 11)
    n = sum(counts)
    r = dad.RotaryPositions(D, device=cuda) if rotate else None
    q, k, v = (torch.randn(lead + n + 5, h, D, generator=g, device=cuda).to(torch.bfloat16) for h in (Hq, Hkv, Hkv))
    part = slice(lead, lead + n)
    want = torch.full_like(q, 9.0)
    dad.kv_cache_append_paged(c, k[part], v[part], starts, q=q[part], q_out=want[part], rotary=r)
    want_pages = c.k.clone(), c.v.clone()
    where = _places(c, ahead, counts)
    for x in (c.k, c.v):
        x[where[0], :, where[1]] = 0
    q_out = torch.full_like(q, 9.0)
    dad.kv_cache_append_paged(c, k, v, starts + lead, q=q, q_out=q_out, rotary=r)
    assert torch.equal(c.k, want_pages[0]) and torch.equal(c.v, want_pages[1]) and torch.equal(q_out, want)
    dad.kv_cache_advance_paged(c, starts + lead, lead + n + 5)
    assert c.lengths.tolist() == [20, 41] and device_status() == 0
