"""GPU: eviction from a KV cache by accumulated attention weight, and the run of calls it belongs to."""
import pytest
import torch

import dadgpt_b200 as dad
from dadgpt_b200.attention import device_status
from tests.cache_reference import attend, check_out, visible
from tests import kernel_ahead

pytestmark = pytest.mark.gpu


def _kept(weights, n, budget, recent):
    """The rows of one head that stay, by sorting in Python."""
    if n <= budget:
        return list(range(n))
    w = weights[:n].tolist()
    # NaN counts as less than everything, -inf too: a NaN comes behind a -inf
    order = sorted(range(n - recent), key=lambda j: (w[j] != w[j], -w[j] if w[j] == w[j] else 0, j))
    return sorted(order[:budget - recent]) + list(range(n - recent, n))


def _made(cuda, B, H, max_len, D, lengths, seed, ties=False):
    g = torch.Generator(device=cuda).manual_seed(seed)
    c = dad.KVCacheBF16(B, H, max_len, D, device=cuda, weights=True)
    c.k.normal_(generator=g)
    c.v.normal_(generator=g)
    c.weights.exponential_(generator=g)
    if ties:
        c.weights.mul_(2).floor_()
        c.weights[:, :, ::7] = -0.0
        c.weights[:, :, 3::11] = float("nan")
        c.weights[:, :, 5::13] = float("inf")
        c.weights[:, :, 6::17] = -1.5
        c.weights[:, :, 8::19] = float("-inf")
    c.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    return c


def _check(dst, src, before, lengths, budget, recent):
    k, v, w, dk, dv, dw = before
    for b, n in enumerate(lengths):
        for h in range(src.H):
            rows = torch.tensor(_kept(w[b, h], n, budget, recent), device=k.device, dtype=torch.long)
            m = len(rows)
            for now, old, to in ((dst.k, k, dk), (dst.v, v, dv), (dst.weights, w, dw)):
                assert torch.equal(now[b, h, :m].view(torch.int16), old[b, h, rows].view(torch.int16))
                assert torch.equal(now[b, h, m:].view(torch.int16), to[b, h, m:].view(torch.int16))
    assert dst.lengths.tolist() == [min(n, budget) for n in lengths]


CASES = [(1, 3, 9000, 64, [8999], 2048, 256), (2, 5, 2500, 128, [2500, 1024], 1024, 0), (7, 3, 300, 64, [0, 1, 63, 64, 65, 300, 299], 64, 64),
         (3, 2, 40, 128, [40, 10, 11], 10, 3), (5, 300, 130, 64, [130, 5, 64, 100, 129], 100, 99), (2, 2, 1030, 64, [1030, 1025], 1, 0),
         (2, 2, 60000, 64, [60000, 50000], 700, 50), (1, 1, 60000, 64, [59999], 40000, 7), (1, 2, 196608, 64, [196608], 1500, 1500)]


@pytest.mark.parametrize("ties", [False, True], ids=["", "ties"])
@pytest.mark.parametrize("place", ["another", "same"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:4])))
def test_what_stays(cuda, case, place, ties):
    B, H, max_len, D, lengths, budget, recent = case
    src = _made(cuda, B, H, max_len, D, lengths, 1, ties)
    dst = src if place == "same" else _made(cuda, B, H, budget + 3, D, [77] * B, 2)
    before = [t.clone() for t in (src.k, src.v, src.weights, dst.k, dst.v, dst.weights)]
    dad.kv_cache_evict_bf16(dst, src, budget, recent)
    _check(dst, src, before, lengths, budget, recent)
    if place == "another":
        assert torch.equal(src.k, before[0]) and torch.equal(src.lengths.cpu(), torch.tensor(lengths, dtype=torch.int32))
    assert device_status() == 0


def test_all_weights_equal_or_not_a_number(cuda):
    src = _made(cuda, 1, 3, 700, 64, [700], 3)
    src.weights[0, 0] = 0.25
    src.weights[0, 1] = float("nan")
    src.weights[0, 2] = 0.0
    src.weights[0, 2, 500] = -0.0
    before = [t.clone() for t in (src.k, src.v, src.weights, src.k, src.v, src.weights)]
    dad.kv_cache_evict_bf16(src, src, 501, 0)
    _check(src, src, before, [700], 501, 0)
    assert torch.equal(src.k[0, :, :501], before[0][0, :, :501])


def test_an_invalid_length_is_left_alone(cuda):
    src = _made(cuda, 3, 4, 50, 64, [50, 51, -1], 4)
    dst = _made(cuda, 3, 4, 50, 64, [9, 9, 9], 5)
    k0 = dst.k.clone()
    dad.kv_cache_evict_bf16(dst, src, 20, 5)
    assert device_status() == -1 and dst.lengths.tolist() == [20, 9, 9] and torch.equal(dst.k[1:], k0[1:])
    k0 = src.k.clone()
    dad.kv_cache_evict_bf16(src, src, 20, 5)
    assert device_status() == -1 and src.lengths.tolist() == [20, 51, -1] and torch.equal(src.k[1:], k0[1:])


@pytest.mark.parametrize("graph", [False, True], ids=["", "graph"])
def test_a_generation_under_a_budget(cuda, graph):
    """Tokens with their weights added up, eviction whenever the budget is passed by 8, against a float64 model of it."""
    B, H, D, max_len, budget, recent, scale = 3, 2, 64, 48, 32, 6, 0.125
    g = torch.Generator(device=cuda).manual_seed(6)
    c = dad.KVCacheBF16(B, H, max_len, D, device=cuda, weights=True)
    rows = [[([], [], []) for _ in range(H)] for _ in range(B)]   # K, V, weight of every head's rows
    q, kn, vn = (torch.zeros(B, H, D, device=cuda, dtype=torch.bfloat16) for _ in range(3))
    out = torch.empty_like(q)

    def step():
        dad.decode_attention_bf16_window(out, q, kn, vn, c, scale, weights=True)

    def evict():
        dad.kv_cache_evict_bf16(c, c, budget, recent)

    run, drop = step, evict
    if graph:
        step()
        evict()
        c.lengths.zero_()
        graphs = []
        for f in (step, evict):
            one = torch.cuda.CUDAGraph()
            with torch.cuda.graph(one):
                f()
            graphs.append(one)
        run, drop = graphs[0].replay, graphs[1].replay
    for token in range(100):
        for x in (q, kn, vn):
            x.copy_(torch.randn(B, H, D, device=cuda, generator=g) * 2)
        run()
        for b in range(B):
            for h in range(H):
                ks, vs, ws = rows[b][h]
                ks.append(kn[b, h].clone())
                vs.append(vn[b, h].clone())
                n = len(ks)
                k, v = torch.stack(ks)[None], torch.stack(vs)[None]
                want, p, bound, largest = attend(q[b, h][None], k, v, visible(n - 1, n, 0, 0), scale)
                check_out(out[b, h][None], want, bound, largest)
                ws.append(0.0)
                rows[b][h] = (ks, vs, [x + y for x, y in zip(ws, p[0].tolist())])
        if len(rows[0][0][0]) == budget + 8:
            drop()
            for b in range(B):
                for h in range(H):
                    ks, vs, ws = rows[b][h]
                    stay = _kept(torch.tensor(ws, dtype=torch.float64), len(ws), budget, recent)
                    rows[b][h] = tuple([x[i] for i in stay] for x in (ks, vs, ws))
                    assert torch.equal(c.k[b, h, :budget], torch.stack(rows[b][h][0]))
            assert c.lengths.tolist() == [budget] * B
    assert device_status() == 0


def test_the_kernel_ahead_may_write_weights_and_lengths(cuda):
    src = _made(cuda, 2, 3, 300, 64, [300, 200], 7)
    want, dst = (_made(cuda, 2, 3, 300, 64, [0, 0], 8) for _ in range(2))
    dad.kv_cache_evict_bf16(want, src, 100, 10)
    for target in (src.weights, src.lengths, src.v):
        source = target.clone()
        target.zero_()
        torch.cuda.synchronize()
        kernel_ahead.launch(target, source)
        dad.kv_cache_evict_bf16(dst, src, 100, 10)
        for x in ("k", "v", "weights", "lengths"):
            assert torch.equal(getattr(dst, x), getattr(want, x))


def test_two_caches_on_two_streams_at_once(cuda):
    """Steps and evictions of two caches, each on its own stream, leave what they leave one after the other."""
    def run(at_once):
        streams = [torch.cuda.Stream(), torch.cuda.Stream()] if at_once else [torch.cuda.current_stream()] * 2
        caches = [_made(cuda, 40, 12, 400, 64, [(b * 7 + 13 * i) % 300 for b in range(40)], 31 + i) for i in range(2)]
        small = [dad.KVCacheFP8(3, 12, 1000, 64, device=cuda) for _ in range(2)]
        g = torch.Generator(device=cuda).manual_seed(33)
        heads = torch.randn(3, 12, 700, 64, device=cuda, generator=g).bfloat16()
        x = torch.randn(2, 4, 40, 12, 64, device=cuda, generator=g).bfloat16()
        torch.cuda.synchronize()
        for _ in range(3):
            for i, (st, c, f) in enumerate(zip(streams, caches, small)):
                with torch.cuda.stream(st):
                    dad.decode_attention_bf16_window(x[i, 3], x[i, 0], x[i, 1], x[i, 2], c, 0.125, weights=True)
                    dad.kv_cache_evict_bf16(c, c, 150, 20)
                    dad.kv_cache_fill_fp8(f, heads, heads)
                    dad.decode_attention_fp8(x[i, 3, :3], x[i, 0, :3], x[i, 1, :3], x[i, 2, :3], f, 0.125)
        torch.cuda.synchronize()
        assert device_status() == 0
        return [t for c, f in zip(caches, small) for t in (c.k, c.v, c.weights, c.lengths, f.k.view(torch.uint8), f.k_tail, f.lengths)] + [x]

    for a, b in zip(run(False), run(True)):
        assert torch.equal(a, b)
