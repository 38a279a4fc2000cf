"""Plain float64 forms of rotary positions and of a paged KV cache, and the bounds that results are held to."""
import math

import torch

import dadgpt_b200 as dad

U = 2.0 ** -24          # half a step of fp32, relative
HALF_BF16 = 2.0 ** -8   # of bf16


def frequencies(rot, base=10000.0, scaling=None, stretch=1.0, trained_len=0, low=1.0, high=32.0):
    """Radians per position from the definition, one pair at a time."""
    got = []
    for i in range(rot // 2):
        b = base * stretch ** (rot / (rot - 2)) if scaling == "base" else base
        w = math.exp(-2.0 * i / rot * math.log(b))
        if scaling == "linear":
            w /= stretch
        if scaling == "parts":
            g = min(1.0, max(0.0, (trained_len * w / (2 * math.pi) - low) / (high - low)))
            w = g * w + (1 - g) * w / stretch
        got.append(w)
    return torch.tensor(got, dtype=torch.float64)


def turn(x, positions, rotary, sign=1):
    """x [..., heads, D] turned by positions [...]: values in float64, and how far fp32 results may be off."""
    f = rotary.freq.to(x.device)
    rot = rotary.rot_dim
    angle = positions.to(x.device).double()[..., None, None] * f
    c, s = rotary.factor * torch.cos(angle), sign * rotary.factor * torch.sin(angle)
    x = x.double()
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if rotary.interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., first], x[..., second]
    y, size = x.clone(), torch.zeros_like(x)
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(rotary.factor)
    return y, size


def check_turned(got, want, size):
    """fp32: the angle's conversion 2^-25.3, sine and cosine 2^-23, three roundings of 2^-24: below 2^-21 of |x1| + |x2|.
    bf16: sine and cosine to 2^-21, below 2^-20 together, and the rounding of the result."""
    if got.dtype == torch.float32:
        allowed = 2.0 ** -21 * size
    else:
        allowed = 2.0 ** -20 * size + HALF_BF16 * (want.abs() + 2.0 ** -20 * size)
    off = (got.double() - want).abs()
    assert bool((off <= allowed).all()), f"off by {off.max().item()}, of {want.abs().max().item()}"


def made(cuda, Hkv, D, page, ahead, counts, seed, extra_pages=3, max_pages=None, garbage=None):
    """A paged cache of sequences with these rows ahead and room for these counts, pages dealt out at random; every row that
    belongs to no sequence is `garbage` (or old values)."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    B = len(ahead)
    need = [-(-(a + n) // page) for a, n in zip(ahead, counts)]
    pages = sum(need) + extra_pages
    c = dad.KVCachePagedBF16(B, Hkv, pages, page, max_pages or max(max(need), 1), D, device=cuda)
    c.k.normal_(generator=g)
    c.v.normal_(generator=g)
    dealt = torch.randperm(pages, generator=g, device=cuda).to(torch.int32)
    used = torch.zeros(pages, page, dtype=torch.bool, device=cuda)
    c.page_table.fill_(-7)   # entries behind a sequence's last row are not read
    at = 0
    for b, n in enumerate(need):
        c.page_table[b, :n] = dealt[at:at + n]
        rows = torch.arange(n * page, device=cuda) < ahead[b] + counts[b]
        if n:
            used[dealt[at:at + n].long()] = rows.view(n, page)
        at += n
    if garbage is not None:
        hole = ~used[:, None, :, None].expand_as(c.k)
        c.k[hole] = garbage
        c.v[hole] = garbage
    c.lengths.copy_(torch.tensor(ahead, dtype=torch.int32))
    starts = torch.tensor([0] + list(counts)).cumsum(0).to(torch.int32).to(cuda)
    return c, starts, g


def rows_of(cache, pool, b, n):
    """The first n rows of sequence b: [H, n, D] in float64."""
    table = cache.page_table[b, :-(-n // cache.page_size)].long()
    return pool[table].transpose(0, 1).flatten(1, 2)[:, :n].double()


def attend(q, k, v, first, scale, q_off=0.0):
    """q [n,H,D] (float64) at rows first .. of k, v [Hkv,rows,D] -> out [n,H,D], lse [n,H], bounds of both.

    A score is a sum of D products in fp32 (D + 2 roundings of 2^-23 of the sum of absolute values, tensor cores may cut off),
    and q may be off by q_off of itself; that moves its exponential and the sum's. Probabilities are rounded to bf16 for the
    product with V, whose sum of n terms adds n roundings; ex2 and the like 2^-21. lse adds its own rounding and log2's."""
    n, H, D = q.shape
    group = H // k.shape[0]
    at = first + torch.arange(n, device=q.device)
    late = torch.arange(k.shape[1], device=q.device) > at[:, None]
    out, lse = torch.empty(n, H, D, dtype=torch.float64, device=q.device), torch.empty(n, H, dtype=torch.float64, device=q.device)
    out_bound, lse_bound = torch.empty_like(out), torch.empty_like(lse)
    for h in range(H):
        K, V = k[h // group], v[h // group]
        s = (q[:, h] @ K.T * scale).masked_fill(late, float("-inf"))
        size = (q[:, h].abs() @ K.abs().T * scale).masked_fill(late, 0.0).amax(1)
        lse[:, h] = torch.logsumexp(s, 1)
        p = torch.exp(s - lse[:, h, None])
        out[:, h] = p @ V
        off = (2 * (D + 2) * U + q_off) * size
        rel = torch.expm1(2 * off) + 4 * (at + 5) * U + 2.0 ** -21
        out_bound[:, h] = (rel + HALF_BF16 * (1 + rel))[:, None] * (p @ V.abs())
        # the sum's exponentials are taken from the first maximum within 2^8: their sum's error is relative
        lse_bound[:, h] = off + 2 * (at + 5) * U + 2.0 ** -21 + 4 * U * lse[:, h].abs() + 2 * U * size
    return out, lse, out_bound + HALF_BF16 * (out.abs() + out_bound), lse_bound


def check(got, want, bound, what="out"):
    off = (got.double() - want).abs()
    good = off <= bound
    assert bool(good.all()), f"{what}: {int((~good).sum())} of {good.numel()} off, the most by {off.nan_to_num(9e9).max().item()}, " \
                             f"{(off / bound).nan_to_num(9e9).max().item()} of the bound, first at {torch.nonzero(~good)[0].tolist()}"
