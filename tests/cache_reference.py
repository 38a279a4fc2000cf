"""Plain float64 forms of the cache operators, and the bounds that their results are held to."""
import torch

BLOCK = 64
U = 2.0 ** -24          # half a step of fp32, relative
HALF_BF16 = 2.0 ** -8   # of bf16


def visible(length, rows, window, sinks):
    """Whether the token at row `length` sees each of rows 0 .. rows - 1."""
    j = torch.arange(rows)
    return (j <= length) & ((length - j < window) | (j < sinks) if window else torch.ones(rows, dtype=torch.bool))


def attend(q, k, v, seen, scale):
    """q [H,D], k, v [H,L,D], seen [L] -> out [H,D], probabilities [H,L] (0 where not seen), bound [H]: how far a
    probability may be off, relative, in fp32 arithmetic of any order: a score is a sum of D products (D + 2 roundings
    of the sum of absolute values, scale and unit among them), which moves its exponential and the sum's; the sum of n
    exponentials and of their products adds n roundings each, ex2 and the divisions a few (2^-21 covers eight)."""
    device = q.device
    at = torch.nonzero(seen).flatten().to(device)
    q, ks, vs = q.double(), k[:, at].double(), v[:, at].double()
    s = torch.einsum("hd,hld->hl", q, ks) * scale
    size = torch.einsum("hd,hld->hl", q.abs(), ks.abs()).amax(1) * abs(scale)
    p = torch.softmax(s, 1)
    out = torch.einsum("hl,hld->hd", p, vs)
    full = torch.zeros(k.shape[:2], dtype=torch.float64, device=device)
    full[:, at] = p
    bound = 2 * (q.shape[1] + 2) * U * size + 2 * (len(at) + 4) * U + 2.0 ** -21
    return out, full, bound, vs.abs().amax((1, 2))


def check_out(got, want, bound, largest):
    """got [H,D] bf16: each probability off by at most `bound` of itself, then one rounding."""
    allowed = bound[:, None] * largest[:, None] + HALF_BF16 * (want.abs() + bound[:, None] * largest[:, None])
    off = (got.double() - want).abs()
    assert bool((off <= allowed).all()), f"off by {off.max().item()}, {(off / allowed).max().item()} of the bound"


_CODES = torch.arange(127, dtype=torch.int64)   # positive e4m3 codes: 0 .. 448


def _code_values():
    e, m = _CODES // 8, _CODES % 8
    return torch.where(e == 0, m.double() / 8 * 2.0 ** -6, (1 + m.double() / 8) * 2.0 ** (e.double() - 7))


def quantise(x):
    """[..., 64, D] (bf16 values) -> codes (uint8), scale [...] in float64, by search in the table of e4m3 numbers."""
    x = x.double().cpu()
    finite = torch.where(torch.isfinite(x), x.abs(), 0.0)
    most = finite.amax((-1, -2))
    mantissa, exponent = torch.frexp(most)
    exponent = torch.where(most > 0, exponent, -126)   # (frexp gives 0 for 0)
    scale = 2.0 ** (exponent - 9 + (mantissa > 0.875).int()).clamp(min=-126).double()   # 448 = 0.875 * 2^9
    y = finite / scale[..., None, None]
    table = _code_values()
    above = torch.searchsorted(table, y).clamp(max=126)
    below = (above - 1).clamp(min=0)
    up, down = table[above] - y, y - table[below]
    code = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    code = torch.where(torch.signbit(x), code + 128, code)
    code = torch.where(torch.isfinite(x), code, 127)
    return code.to(torch.uint8), scale


def values(codes, scale):
    """The numbers that codes [..., 64, D] stand for."""
    c = codes.cpu().long()
    v = torch.cat([_code_values(), torch.full((1,), float("nan"), dtype=torch.float64)])[c % 128]
    return torch.where(c >= 128, -v, v) * scale.cpu().double()[..., None, None]


def cache_rows(cache, b, n):
    """The first n rows of sequence b of an 8-bit cache as float64 K, V [H,n,D] on the cache's device."""
    whole = n // BLOCK
    got = []
    for data, scales, tail in ((cache.k, cache.k_scale, cache.k_tail), (cache.v, cache.v_scale, cache.v_tail)):
        codes = data.view(torch.uint8)[b, :, :whole * BLOCK].unflatten(1, (whole, BLOCK))
        blocks = values(codes, scales[b, :, :whole]).flatten(1, 2)
        got.append(torch.cat([blocks.to(data.device), tail[b, :, :n - whole * BLOCK].double()], 1))
    return got
