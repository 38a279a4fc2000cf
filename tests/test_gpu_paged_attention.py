"""GPU: attention of a packed batch's new tokens over a paged KV cache, against float64, and the run of calls around it."""
import pytest
import torch

import dadgpt_b200 as dad
from dadgpt_b200.attention import device_status
from tests.paged_reference import HALF_BF16, attend, check, made, rows_of, turn

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")

# Hq, Hkv, D, page, rows ahead, new rows
CASES = [(1, 1, 64, 16, [0], [1]), (1, 1, 128, 16, [0], [2]), (12, 12, 64, 16, [700], [301]), (4, 4, 128, 128, [0], [128]),
         (4, 4, 128, 64, [1], [127]), (2, 2, 64, 32, [127, 128, 129], [129, 1, 255]), (8, 2, 128, 64, [5000, 17], [33, 300]),
         (32, 8, 128, 64, [300, 0, 1000], [1, 700, 0]), (6, 2, 64, 32, [0, 95, 0, 40], [0, 96, 257, 0]), (71, 1, 64, 128, [200, 127], [5, 1]),
         (128, 1, 128, 1024, [1023], [3]), (100, 1, 64, 16, [10], [30]), (5, 5, 64, 16, [33] * 100, [i % 5 for i in range(100)]),
         (24, 3, 128, 32, [60, 2000, 31, 32], [500, 100, 1, 32]), (8, 8, 128, 64, [0] * 40, [130] * 40), (12, 12, 64, 64, [0] * 16, [400] * 16),
         (2, 1, 64, 256, [60000], [40]), (3, 3, 128, 16, [255, 256], [1, 257]), (7, 7, 64, 64, [0] * 70, list(range(1, 71)))]


def _check(c, out, lse, q, ahead, counts, scale, sequences=None, q_off=0.0):
    at = 0
    for b, (a, n) in enumerate(zip(ahead, counts)):
        if n and (sequences is None or b in sequences):
            o, s, ob, sb = attend(q[at:at + n].double(), rows_of(c, c.k, b, a + n), rows_of(c, c.v, b, a + n), a, scale, q_off)
            check(out[at:at + n], o, ob, f"out of sequence {b}")
            if lse is not None:
                check(lse[at:at + n], s, sb, f"lse of sequence {b}")
        at += n


@pytest.mark.parametrize("garbage", [None, NAN], ids=["old rows", "nan"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:4])) + f"-{sum(c[5])}")
def test_chunk(cuda, case, garbage):
    Hq, Hkv, D, page, ahead, counts = case
    scale, T = D ** -0.5, sum(counts)
    c, starts, g = made(cuda, Hkv, D, page, ahead, counts, 31, garbage=garbage)
    behind = 3   # rows of nobody
    q = torch.randn(T + behind, Hq, D, generator=g, device=cuda).to(torch.bfloat16)
    out = torch.full_like(q, 9.0)
    lse = torch.full((T + behind, Hq), 9.0, device=cuda)
    k0 = c.k.clone()
    dad.paged_attention_bf16(out, q, c, starts, max(counts), scale, lse=lse)
    many = len(counts) > 20
    _check(c, out, lse, q, ahead, counts, scale, {0, 1, len(counts) // 2, len(counts) - 1} if many else None)
    assert bool((out[T:] == 9.0).all()) and bool((lse[T:] == 9.0).all()) and bool((out[:T] != 9.0).any(-1).all())
    assert device_status() == 0 and torch.equal(c.k.view(torch.int16), k0.view(torch.int16))
    again = torch.empty_like(out)
    dad.paged_attention_bf16(again, q, c, starts, max(counts), scale)   # without lse, and again: the same bits
    assert torch.equal(again[:T], out[:T])


@pytest.mark.parametrize("D", [64, 128])
def test_extreme_values(cuda, D):
    """Scores far apart (accumulators are rescaled), and keys of the new rows themselves."""
    ahead, counts = [200, 130], [260, 7]
    c, starts, g = made(cuda, 2, D, 16, ahead, counts, 32)
    q = torch.randn(sum(counts), 4, D, generator=g, device=cuda).to(torch.bfloat16)
    for b in range(2):
        for i in range(-(-(ahead[b] + counts[b]) // 16)):
            c.k[c.page_table[b, i].long()] *= 1.0 + 0.8 * i       # ever larger scores
    out, lse = torch.empty_like(q), torch.empty(sum(counts), 4, device=cuda)
    dad.paged_attention_bf16(out, q, c, starts, 260, 0.5, lse=lse)
    _check(c, out, lse, q, ahead, counts, 0.5)


def test_strides(cuda):
    Hq, Hkv, D, page, ahead, counts = 6, 2, 128, 32, [50, 0, 333], [140, 61, 1]
    T = sum(counts)
    c, starts, g = made(cuda, Hkv, D, page, ahead, counts, 33)
    fused = torch.randn(T, Hq + 2 * Hkv, D, generator=g, device=cuda).to(torch.bfloat16)
    q = fused[:, :Hq]
    want = torch.empty(T, Hq, D, dtype=torch.bfloat16, device=cuda)
    dad.paged_attention_bf16(want, q.contiguous(), c, starts, 140, 0.125)
    out = torch.full((Hq, T + 1, D + 8), 9.0, dtype=torch.bfloat16, device=cuda)
    dad.paged_attention_bf16(out[:, 1:, 8:].transpose(0, 1), q, c, starts, 140, 0.125)
    assert torch.equal(out[:, 1:, 8:].transpose(0, 1), want)
    assert bool((out[:, 0] == 9.0).all()) and bool((out[:, :, :8] == 9.0).all())
    heads = q.transpose(0, 1).contiguous()   # [H, T, D]
    dad.paged_attention_bf16(out[:, 1:, 8:].transpose(0, 1), heads.transpose(0, 1), c, starts, 140, 0.125)
    assert torch.equal(out[:, 1:, 8:].transpose(0, 1), want)
    with pytest.raises(RuntimeError, match="over each other"):
        dad.paged_attention_bf16(want, q[:, :1].expand(T, Hq, D), c, starts, 140, 0.125)
    with pytest.raises(RuntimeError, match="multiple"):
        dad.paged_attention_bf16(want[:, :5], q[:, :5], c, starts, 140, 0.125)
    with pytest.raises(ValueError, match="lse"):
        dad.paged_attention_bf16(want, q, c, starts, 140, 0.125, lse=torch.empty(T, Hq - 1, device=cuda))
    with pytest.raises(ValueError, match="starts"):
        dad.paged_attention_bf16(want, q, c, starts[:-1], 140, 0.125)


@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])   # clusters, and pairs of tiles
@pytest.mark.parametrize("what", ["negative length", "no room", "page", "falling starts", "more than max_new"])
def test_a_sequence_that_does_not_fit_is_left_alone(cuda, what, many):
    H = 40 if many else 2
    ahead, counts = [40, 300, 7], [200, 150, 20]
    c, starts, g = made(cuda, H, 64, 16, ahead, counts, 34, max_pages=30)
    T, max_new = sum(counts), 200
    q = torch.randn(T, H, 64, generator=g, device=cuda).to(torch.bfloat16)
    left = slice(200, 350)
    if what == "negative length":
        c.lengths[1] = -5
    elif what == "no room":
        c.lengths[1] = 480 - 149
    elif what == "page":
        c.page_table[1, 2] = c.pages
    elif what == "more than max_new":
        max_new, left = 150, slice(0, 200)
    else:
        starts[2] = 199
        left = slice(350, 350)
    out = torch.full_like(q, 9.0)
    dad.paged_attention_bf16(out, q, c, starts, max_new, 0.125)
    assert device_status() == -1 and device_status() == 0
    if what == "falling starts":   # (sequence 2 then has rows 199 .., more than max_new or not its own; sequence 0 is whole)
        return
    assert bool((out[left] == 9.0).all())
    sequences = {0, 1, 2} - ({0} if what == "more than max_new" else {1})
    _check(c, out, None, q, ahead, counts, 0.125, sequences)


def test_pieces_of_prompts_then_single_tokens(cuda):
    """The life of a batch: prompts in pieces, turned, appended and attended for, then decode steps, on pages that are dealt
    out as sequences grow, through two layers that share table and lengths. Against float64 over whole sequences."""
    Hq, Hkv, D, page, scale = 8, 2, 64, 16, 0.125
    total, B = [300, 77, 190], 3
    r = dad.RotaryPositions(D, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(40)
    first = dad.KVCachePagedBF16(B, Hkv, 60, page, 20, D, device=cuda)
    layers = [first, dad.KVCachePagedBF16(B, Hkv, 60, page, 20, D, device=cuda, page_table=first.page_table, lengths=first.lengths)]
    data = [[[torch.randn(n, h, D, generator=g, device=cuda).to(torch.bfloat16) for h in (Hq, Hkv, Hkv)] for n in total] for _ in layers]
    got = [[[] for _ in total] for _ in layers]
    free = list(torch.randperm(60, generator=torch.Generator().manual_seed(1)).tolist())
    have, taken = [0] * B, [0] * B
    steps = [[100, 5, 0], [150, 70, 1], [0, 0, 187], [48, 0, 0]]
    steps += [[1 if have_ < t else 0 for have_, t in zip([298, 75, 188], total)]] * 2
    for counts in steps:
        single = counts == [1, 1, 1]
        for b in range(B):
            while taken[b] * page < have[b] + counts[b]:
                first.page_table[b, taken[b]] = free.pop()
                taken[b] += 1
        starts = torch.tensor([0] + counts).cumsum(0).to(torch.int32).to(cuda)
        for layer, c in enumerate(layers):
            q, k, v = (torch.cat([data[layer][b][i][have[b]:have[b] + counts[b]] for b in range(B)]) for i in range(3))
            out = torch.empty_like(q)
            if single:
                dad.decode_attention_paged_bf16(out, q, k, v, c, scale, rotary=r)
            else:
                dad.kv_cache_append_paged(c, k, v, starts, q=q, q_out=q, rotary=r)
                dad.paged_attention_bf16(out, q, c, starts, max(counts), scale)
            at = 0
            for b in range(B):
                got[layer][b].append(out[at:at + counts[b]])
                at += counts[b]
        have = [h + n for h, n in zip(have, counts)]
        if single:
            dad.kv_cache_advance_paged(first)
        else:
            dad.kv_cache_advance_paged(first, starts, sum(counts))
    assert have == total and first.lengths.tolist() == total and device_status() == 0
    for layer, c in enumerate(layers):
        for b, n in enumerate(total):
            at = torch.arange(n, device=cuda)
            q = turn(data[layer][b][0], at, r)[0]
            o, _, ob, _ = attend(q, rows_of(c, c.k, b, n), rows_of(c, c.v, b, n), 0, scale, HALF_BF16 + 2.0 ** -19)
            check(torch.cat(got[layer][b]), o, ob, f"layer {layer}, sequence {b}")
            # and the fused causal attention of the whole prompt on the same turned queries and keys
            if layer == 0:
                heads = [x.bfloat16().contiguous() for x in (q.transpose(0, 1), rows_of(c, c.k, b, n).repeat_interleave(Hq // Hkv, 0),
                                                             rows_of(c, c.v, b, n).repeat_interleave(Hq // Hkv, 0))]
                whole, lse = torch.empty_like(heads[0]), torch.empty(Hq, n, device=cuda)
                dad.gpu_flash_attention_forward_bf16(whole, lse, *heads, Hq, n, D, scale)
                assert float((torch.cat(got[layer][b]).transpose(0, 1).float() - whole.float()).abs().max()) <= 2e-2


def test_captured_and_on_two_streams(cuda):
    cases = [(made(cuda, 2, 128, 64, [900, 10], [60, 300], 50)), (made(cuda, 2, 128, 64, [0, 2000], [500, 1], 51))]
    qs, want, got = [], [], []
    for c, starts, g in cases:
        T = int(starts[-1])
        qs.append(torch.randn(T, 8, 128, generator=g, device=cuda).to(torch.bfloat16))
        want.append(torch.empty_like(qs[-1]))
        got.append(torch.empty_like(qs[-1]))
        dad.paged_attention_bf16(want[-1], qs[-1], c, starts, 500, 0.1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    graphs = [torch.cuda.CUDAGraph() for _ in cases]
    for i, (c, starts, _) in enumerate(cases):
        with torch.cuda.graph(graphs[i], stream=streams[i]):
            dad.paged_attention_bf16(got[i], qs[i], c, starts, 500, 0.1)
    for _ in range(4):
        for i, (c, starts, _) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].zero_()
                graphs[i].replay()
                dad.paged_attention_bf16(got[i], qs[i], c, starts, 500, 0.1)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(got[i], want[i])
    assert device_status() == 0


def test_rows_beyond_31_bits_of_bytes(cuda):
    """A pool whose rows lie beyond 2^32 bytes and 2^31 elements."""
    H, D, page = 8, 128, 64
    pages = 2 ** 32 // (H * D * page) + 40
    c = dad.KVCachePagedBF16(1, H, pages, page, 8, D, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(60)
    last = torch.arange(pages - 5, pages, device=cuda, dtype=torch.int32)
    c.page_table[0, :5] = last.flip(0)
    n = 270
    q, k, v = (torch.randn(n, h, D, generator=g, device=cuda).to(torch.bfloat16) for h in (H, H, H))
    starts = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    dad.kv_cache_append_paged(c, k, v, starts)
    assert torch.equal(rows_of(c, c.k, 0, n), k.double().transpose(0, 1)) and not bool(c.k[:pages - 5].any())
    out = torch.empty_like(q)
    dad.paged_attention_bf16(out, q, c, starts, n, 0.09)
    _check(c, out, None, q, [0], [n], 0.09)
    dad.kv_cache_advance_paged(c, starts, n)
    dad.decode_attention_paged_bf16(out[:1], q[:1], k[:1], v[:1], c, 0.09)
    o, _, ob, _ = attend(q[:1].double(), rows_of(c, c.k, 0, n + 1), rows_of(c, c.v, 0, n + 1), n, 0.09)
    check(out[:1], o, ob)
    assert device_status() == 0


@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_rows_ahead_of_the_first_sequence_belong_to_nobody(cuda, many):
    ahead, counts, lead = ([30, 200], [50, 1], 19) if not many else ([30, 200] * 40, [150, 1] * 40, 301)
    c, starts, g = made(cuda, 2, 64, 16, ahead, counts, 41)
    n = sum(counts)
    q = torch.randn(lead + n + 3, 4, 64, generator=g, device=cuda).to(torch.bfloat16)
    part = slice(lead, lead + n)
    want, out = torch.full_like(q, 9.0), torch.full_like(q, 9.0)
    dad.paged_attention_bf16(want[part], q[part], c, starts, max(counts), 0.125)
    dad.paged_attention_bf16(out, q, c, starts + lead, max(counts), 0.125)
    assert torch.equal(out, want) and bool((want[part] != 9.0).any(-1).all()) and device_status() == 0


@pytest.mark.parametrize("D", [64, 128])
def test_many_sequences(cuda, D):
    """Every CTA goes through items of many sequences, some without new tokens, one that does not fit."""
    B, g = 500, torch.Generator().manual_seed(70)
    ahead = torch.randint(0, 200, (B,), generator=g).tolist()
    counts = [0 if b % 7 == 3 else 150 if b % 40 == 0 else 1 + b % 20 for b in range(B)]
    c, starts, gen = made(cuda, 4, D, 16, ahead, counts, 71)
    q = torch.randn(sum(counts), 8, D, generator=gen, device=cuda).to(torch.bfloat16)
    out = torch.full_like(q, 9.0)
    dad.paged_attention_bf16(out, q, c, starts, 150, 0.125)
    assert device_status() == 0 and bool((out != 9.0).any(-1).all())
    _check(c, out, None, q, ahead, counts, 0.125, set(range(0, B, 23)) | {1, B - 1})
    refused = 321
    c.lengths[refused] = -1
    again = torch.full_like(q, 9.0)
    dad.paged_attention_bf16(again, q, c, starts, 150, 0.125)
    assert device_status() != 0
    rows = slice(int(starts[refused]), int(starts[refused + 1]))
    assert bool((again[rows] == 9.0).all())
    again[rows] = out[rows]
    assert torch.equal(again, out)
