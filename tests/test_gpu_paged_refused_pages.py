"""GPU: attention over a paged KV cache with pages outside the pool: which rows are left untouched, and which are not."""
import pytest
import torch

import dadgpt_b200 as dad
from dadgpt_b200.attention import device_status
from tests.paged_reference import made

pytestmark = pytest.mark.gpu


def _run(q, c, starts, max_new):
    out, lse = torch.full_like(q, 9.0), torch.full(q.shape[:2], 9.0, device=q.device)
    dad.paged_attention_bf16(out, q, c, starts, max_new, 0.125, lse=lse)
    return out, lse


def _check(q, c, starts, max_new, untouched):
    """The rows `untouched` (a mask over the packed tokens) keep what they held, the others get what they get without bad pages,
    bit for bit; several times over, since it was once a matter of time."""
    table = c.page_table.clone()
    c.page_table.clamp_(0, c.pages - 1)
    want, want_lse = _run(q, c, starts, max_new)
    assert device_status() == 0 and bool((want != 9.0).any(-1).all())
    c.page_table.copy_(table)
    want[untouched], want_lse[untouched] = 9.0, 9.0
    for _ in range(5):
        out, lse = _run(q, c, starts, max_new)
        assert device_status() == -1
        wrong = ((out != want).any(-1) | (lse != want_lse)).any(1)
        assert not bool(wrong.any()), f"tokens {torch.nonzero(wrong).flatten().tolist()[:20]}"


# One key tile or less: the second group of a tile that the groups share has no steps, or one
@pytest.mark.parametrize("keys", [(1, 60), (65, 128), (1, 128), (129, 256)], ids=lambda k: f"{k[0]}-{k[1]} keys")
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (12, 4)])
@pytest.mark.parametrize("D", [64, 128])
def test_many_short_sequences(cuda, D, Hq, Hkv, keys):
    B, page = 600, 16
    g = torch.Generator().manual_seed(80)
    total = torch.randint(keys[0], keys[1] + 1, (B,), generator=g).tolist()
    counts = [1 + int(torch.randint(0, min(t, 40), (1,), generator=g)) for t in total]
    ahead = [t - n for t, n in zip(total, counts)]
    c, starts, gen = made(cuda, Hkv, D, page, ahead, counts, 81)
    q = torch.randn(sum(counts), Hq, D, generator=gen, device=cuda).to(torch.bfloat16)
    c.page_table.clamp_(0, c.pages - 1)
    untouched = torch.zeros(sum(counts), dtype=torch.bool, device=cuda)
    at = [0] + torch.tensor(counts).cumsum(0).tolist()
    for i, b in enumerate(range(4, B, 9)):   # its first page, its last, its only one
        c.page_table[b, (total[b] - 1) // page if i % 2 else 0] = c.pages if i % 3 else -1
        untouched[at[b]:at[b + 1]] = True
    _check(q, c, starts, max(counts), untouched)


# The first query tile's 128 rows see keys 0 .. 227, the second's 72 keys 0 .. 299
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,H", [(24, 32), (16, 2), (3, 1)], ids=["pairs", "single tiles", "clusters"])
def test_tiles_that_do_not_read_the_page(cuda, B, H, D):
    page, ahead, n = 16, 100, 200
    c, starts, g = made(cuda, H, D, page, [ahead] * B, [n] * B, 82)
    q = torch.randn(B * n, H, D, generator=g, device=cuda).to(torch.bfloat16)
    c.page_table.clamp_(0, c.pages - 1)
    untouched = torch.zeros(B * n, dtype=torch.bool, device=cuda)
    for b, (key, first) in enumerate([(256, 128), (0, 0), (299, 128), (240, 0), (127, 0)][:B]):
        if b < 2 or B > 3:
            c.page_table[b, key // page] = c.pages + 3
            untouched[b * n + first:(b + 1) * n] = True
    _check(q, c, starts, n, untouched)
