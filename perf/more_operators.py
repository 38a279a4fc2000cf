"""Rotary positions and attention over a paged KV cache, as cases whose speed is followed.

Kinds of case (``kind``):
  rotary   queries and keys of a training step turned by their positions, and the gradients turned back
  append   the new tokens of a packed batch written to the pages of their sequences, keys (and queries) turned on the way
  chunk    causal attention of a packed batch's new tokens over all rows of their sequences' pages
  decode   one token for every sequence: turned, appended and attended for in one call

Activations are i.i.d. normal values: after layer norm and a projection they are close to that. Buffers for results and
caches are made once, as a model's arena does. Pages are dealt out in random order, as they are after a while of serving,
and hold old values behind a sequence's last row.
"""
from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _case(name, **c):
    return {"name": name, **c} if name else c


def _rotary(name, B, S, H, Hkv, D, rot, interleaved, dtype, layout, scaling="none", first=0):
    """layout: "heads" [B,H,S,D] as the attention kernels take them, "tokens" [B,S,H,D] as the projections leave them."""
    return _case(name, kind="rotary", B=B, S=S, H=H, Hkv=Hkv, D=D, rot=rot, interleaved=interleaved, dtype=dtype,
                 layout=layout, scaling=scaling, first=first)


def _paged(kind, name, B, H, Hkv, D, page, longest, new, rot, batch="pieces", interleaved=False, dtype="bf16", scaling="none"):
    """B sequences that end up to `longest` rows long, the first one `longest`; rot = 0: no rotation. Of a sequence's rows
    these are this call's, by `batch`: "pieces" a quarter of `new` and more, the first one's `new`; "mixed" the same of
    every third sequence, one row of the others; "prompts" all (new = longest)."""
    return _case(name, kind=kind, B=B, H=H, Hkv=Hkv, D=D, page=page, longest=longest, new=new, rot=rot, batch=batch,
                 interleaved=interleaved, dtype=dtype, scaling=scaling)


def listed():
    return [
        # a short fp32 step on an odd number of tokens
        _rotary("rotary_f32_ragged", 2, 70, 4, 4, 32, 32, False, "f32", "tokens"),
        # GPT-2 124M's shape, batch 16, at full context, heads split
        _rotary("rotary_gpt2_b16", 16, 1024, 12, 12, 64, 64, False, "bf16", "heads"),
        # long context, shared key heads, a part of the head, stretched positions, straight from the projections
        _rotary("rotary_long_part", 1, 8192, 32, 8, 128, 64, True, "bf16", "tokens", "parts", 100000),
        # one user's prompt of odd length from fp32 heads, learned positions: a prefill's rows into pages
        _paged("append", "append_prompt", 1, 12, 12, 64, 16, 301, 301, 0, dtype="f32"),
        # a packed batch of ragged prompts behind a common start, turned
        _paged("append", "append_batch", 16, 32, 8, 128, 64, 4096, 1500, 128),
        # the next piece of one user's prompt
        _paged("chunk", "chunk_one", 1, 12, 12, 64, 16, 1001, 301, 0),
        # serving: single tokens of most sequences beside the prompts of some
        _paged("chunk", "chunk_mixed", 24, 32, 8, 128, 64, 4000, 512, 0, "mixed"),
        # GPT-2 124M's shape: 16 prompts at once, nothing ahead of them
        _paged("chunk", "chunk_prompts", 16, 12, 12, 64, 64, 1024, 1024, 0, "prompts"),
        # the last piece of a long document
        _paged("chunk", "chunk_long", 1, 32, 8, 128, 64, 16384, 2048, 0),
        # DadGPT's own generation loop, one sequence: latency is what counts
        _paged("decode", "decode_paged_one", 1, 12, 12, 64, 16, 700, 1, 64),
        # serving, 64 sequences of mixed length
        _paged("decode", "decode_paged_64seq", 64, 12, 12, 64, 64, 1024, 1, 0),
        # a few long conversations on a model with shared key heads
        _paged("decode", "decode_paged_8seq_long", 8, 32, 8, 128, 64, 16000, 1, 128, scaling="parts"),
    ]


def _log_int(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    kind = rng.choice(["rotary", "append", "chunk", "chunk", "decode", "decode"])
    interleaved = rng.random() < 0.5
    scaling = rng.choice(["none", "none", "linear", "base", "parts"])
    if kind == "rotary":
        D = rng.choice([32, 64, 96, 128])
        Hkv = rng.randint(1, 12)
        H = Hkv * rng.choice([1, 1, 2, 4])
        S = _log_int(rng, 16, 8192)
        B = _log_int(rng, 1, 16)
        dtype = rng.choice(["bf16", "bf16", "f32"])
        while B * S * (H + Hkv) * D * TYPES[dtype].itemsize > 8192 * 40 * 128 * 2:
            B, S = max(1, B // 2), (S if B > 1 else S * 2 // 3)
        rot = rng.choice([D, D, D // 2 // 16 * 16 or 16])
        return _rotary(None, B, S, H, Hkv, D, rot, interleaved, dtype,
                       rng.choice(["heads", "tokens"]), scaling, rng.choice([0, 0, rng.randint(1, 1000000)]))
    D = rng.choice([64, 128])
    Hkv = rng.randint(1, 12)
    group = rng.choice([1, 1, 2, 4, 8, rng.randint(1, 8)])
    page = rng.choice([16, 32, 64, 128])
    longest = _log_int(rng, 100, 16000)
    B = _log_int(rng, 1, 64)
    while B * Hkv * longest * D > 8 * 8 * 16000 * 128 // 2:
        longest, B = (longest // 2 if longest > 400 else longest), max(1, B // 2)
    rot = rng.choice([0, D, D, D // 2])
    if kind == "decode":
        return _paged(kind, None, B, Hkv * group, Hkv, D, page, longest, 1, rot, "pieces", interleaved, "bf16", scaling)
    new = min(longest, _log_int(rng, 2, 4096))
    while B * Hkv * group * new * longest * D > 32 * 2048 * 16384 * 128 // 2 or B * new * (group + 2) * Hkv * D > 40e6:
        new, B = max(2, new // 2), max(1, B // 2)
    batch = rng.choice(["pieces", "mixed", "prompts"])
    if batch == "prompts":
        longest = new
    if kind == "append":
        return _paged(kind, None, B, Hkv * group, Hkv, D, page, longest, new, rot, batch, interleaved,
                      rng.choice(["bf16", "f32"]), scaling)
    return _paged(kind, None, B, Hkv * group, Hkv, D, page, longest, new, 0, batch)


class _State:
    pass


class _Cache:
    """What the paged cache below has in common with the framework's: tensors and sizes."""

    def __init__(self, B, H, pages, page_size, max_pages, D):
        self.B, self.H, self.pages, self.page_size, self.max_pages, self.D = B, H, pages, page_size, max_pages, D
        self.k = torch.zeros(pages, H, page_size, D, dtype=torch.bfloat16, device="cuda")
        self.v = torch.zeros_like(self.k)
        self.page_table = torch.zeros(B, max_pages, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(B, dtype=torch.int32, device="cuda")


SCALINGS = {"none": dict(), "linear": dict(scaling="linear", stretch=4.0), "base": dict(scaling="base", stretch=8.0),
            "parts": dict(scaling="parts", stretch=16.0, trained_len=4096, low=1.0, high=32.0)}


def _sizes(case):
    """(rows ahead of this call, rows of this call) for each sequence, as a program's scheduler knows them: the same for
    every seed, so that outputs have the same shapes."""
    B, longest, new = case["B"], case["longest"], case["new"]
    rng = random.Random(1000 * B + longest)
    ends = [1 + int((b + rng.random()) * longest / B) for b in range(B)]   # one in each of B equal parts of 1..longest
    rng.shuffle(ends)
    ends = [longest] + [min(n, longest) for n in ends[1:]]
    if case["kind"] == "decode":
        return [n - 1 for n in ends], [1] * B
    counts = [new]
    for b in range(1, B):
        piece = max(1, min(ends[b], int(new * (0.25 + 0.75 * rng.random()))))
        counts.append(ends[b] if case["batch"] == "prompts" else 1 if case["batch"] == "mixed" and b % 3 else piece)
    return [n - c for n, c in zip(ends, counts)], counts


def _values(g, dtype, *shape):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, 1.0, generator=g)


def prepare(case, seed):
    s = _State()
    s.case = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    dtype = TYPES[case["dtype"]]
    s.scale = D ** -0.5
    s.rotary = None
    if case["rot"] and own:
        import dadgpt_b200 as dad
        s.rotary = dad.RotaryPositions(case["rot"], base=10000.0, interleaved=case["interleaved"], **SCALINGS[case["scaling"]])
    if case["kind"] == "rotary":
        B, S = case["B"], case["S"]

        def tensor(heads):   # [B,S,heads,D] however it lies in memory
            if case["layout"] == "heads":
                return _values(g, dtype, B, heads, S, D).transpose(1, 2)
            return _values(g, dtype, B, S, heads, D)

        s.q, s.k, s.dq_turned, s.dk_turned = tensor(H), tensor(Hkv), tensor(H), tensor(Hkv)
        s.q_turned, s.k_turned, s.dq, s.dk = (torch.empty_like(x) for x in (s.q, s.k, s.q, s.k))
        return s
    B, page = case["B"], case["page"]
    s.ahead, s.counts = _sizes(case)
    need = [-(-(a + c) // page) for a, c in zip(s.ahead, s.counts)]
    pages, max_pages = sum(need) + 1, -(-case["longest"] // page)
    if own:
        import dadgpt_b200 as dad
        s.cache = dad.KVCachePagedBF16(B, Hkv, pages, page, max_pages, D)
    else:
        s.cache = _Cache(B, Hkv, pages, page, max_pages, D)
    c = s.cache
    c.k.normal_(generator=g)
    c.v.normal_(generator=g)
    dealt = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    at = 0
    for b, n in enumerate(need):
        c.page_table[b, :n] = dealt[at:at + n]
        at += n
    c.lengths.copy_(torch.tensor(s.ahead, dtype=torch.int32))
    s.T = sum(s.counts)
    s.starts = torch.tensor([0] + s.counts).cumsum(0).to(torch.int32).cuda()
    s.q = _values(g, dtype, s.T, H, D)
    if case["kind"] != "chunk":
        s.k_new, s.v_new = _values(g, dtype, s.T, Hkv, D), _values(g, dtype, s.T, Hkv, D)
    if case["kind"] == "append":
        s.q_out = torch.empty(s.T, H, D, dtype=torch.bfloat16, device="cuda") if case["rot"] else None
    else:
        s.out = torch.empty_like(s.q)
        s.lse = torch.empty(s.T, H, device="cuda")
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------

def _frequencies(case):
    """Radians per position of each pair, float64, and the factor of the rotated part."""
    rot, how = case["rot"], SCALINGS[case["scaling"]]
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    base, stretch = 10000.0, how.get("stretch", 1.0)
    if case["scaling"] == "base":
        base *= stretch ** (rot / max(rot - 2, 1))
    f = base ** (-2.0 * i / rot)
    if case["scaling"] == "linear":
        f = f / stretch
    if case["scaling"] == "parts":
        turns = how["trained_len"] * f / (2 * math.pi)
        keep = ((turns - how["low"]) / (how["high"] - how["low"])).clamp(0, 1)
        f = f * keep + f / stretch * (1 - keep)
        return f, 0.1 * math.log(stretch) + 1
    return f, 1.0


def _turn(x, positions, case, back=False):
    """x [..., heads, D] turned by positions [...] in 32 bits, angles in 64."""
    rot = case["rot"]
    f, factor = _frequencies(case)
    angle = positions.double()[..., None, None] * f
    c, s = (torch.cos(angle) * factor).float(), (torch.sin(angle) * factor).float()
    if back:
        s = -s
    x = x.float()
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _token_rows(s):
    """(sequence, row in the sequence) of every new token, on the GPU."""
    t = torch.arange(s.T, device="cuda")
    b = torch.searchsorted(s.starts[1:].long(), t, right=True)
    return b, s.cache.lengths.long()[b] + t - s.starts.long()[b]


def _append_plain(s, q_out):
    c, case = s.cache, s.case
    b, row = _token_rows(s)
    k = _turn(s.k_new, row, case) if case["rot"] else s.k_new.float()
    if q_out is not None:
        q_out.copy_(_turn(s.q, row, case))
    at = c.page_table[b, row // c.page_size].long()
    c.k[at, :, row % c.page_size] = k.to(torch.bfloat16)
    c.v[at, :, row % c.page_size] = s.v_new.to(torch.bfloat16)


def _gathered(pool, table, n):
    """The first n rows of a sequence: [heads, n, D] in 32 bits."""
    x = pool[table.long()]                                       # [pages, heads, page, D]
    return x.transpose(0, 1).flatten(1, 2)[:, :n].float()


def _chunk_plain(s):
    c, case = s.cache, s.case
    group = case["H"] // case["Hkv"]
    at = 0
    for b, (ahead, n) in enumerate(zip(s.ahead, s.counts)):
        rows = ahead + n
        table = c.page_table[b, :-(-rows // c.page_size)]
        k, v = _gathered(c.k, table, rows), _gathered(c.v, table, rows)
        hidden = torch.arange(rows, device="cuda") > torch.arange(ahead, rows, device="cuda")[:, None]
        for h in range(case["Hkv"]):
            q = s.q[at:at + n, h * group:(h + 1) * group].float().transpose(0, 1)          # [group, n, D]
            scores = (q @ k[h].T).mul_(s.scale).masked_fill_(hidden, float("-inf"))
            lse = torch.logsumexp(scores, -1)
            out = scores.sub_(lse[..., None]).exp_() @ v[h]
            s.out[at:at + n, h * group:(h + 1) * group] = out.transpose(0, 1)
            s.lse[at:at + n, h * group:(h + 1) * group] = lse.T
        at += n


def _decode_plain(s):
    c, case = s.cache, s.case
    q = _turn(s.q, c.lengths, case) if case["rot"] else s.q.float()
    _append_plain(s, None)
    group, n = case["H"] // case["Hkv"], c.lengths.long()
    seen = torch.arange(c.max_pages * c.page_size, device="cuda") <= n[:, None]            # [B, rows]
    for h in range(case["Hkv"]):
        k = c.k[:, h][c.page_table.long()].flatten(1, 2).float()                            # [B, rows, D]
        v = c.v[:, h][c.page_table.long()].flatten(1, 2).float()
        scores = (q[:, h * group:(h + 1) * group] @ k.mT) * s.scale
        scores = scores.masked_fill_(~seen[:, None], float("-inf"))
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        v = v.masked_fill_(~seen[..., None], 0.0)
        s.out[:, h * group:(h + 1) * group] = (p @ v) / p.sum(-1, keepdim=True)


# ---- one pass ---------------------------------------------------------------------------------------------------

def run(s):
    case, kind = s.case, s.case["kind"]
    if own:
        import dadgpt_b200 as dad
    if kind == "rotary":
        if own:
            dad.rotary_forward(s.q_turned, s.k_turned, s.q, s.k, s.rotary, first=case["first"])
            dad.rotary_backward(s.dq, s.dk, s.dq_turned, s.dk_turned, s.rotary, first=case["first"])
        else:
            at = torch.arange(case["first"], case["first"] + case["S"], device="cuda")
            s.q_turned.copy_(_turn(s.q, at, case))
            s.k_turned.copy_(_turn(s.k, at, case))
            s.dq.copy_(_turn(s.dq_turned, at, case, back=True))
            s.dk.copy_(_turn(s.dk_turned, at, case, back=True))
        return s.q_turned, s.k_turned, s.dq, s.dk
    c = s.cache
    if kind == "append":
        if own:
            dad.kv_cache_append_paged(c, s.k_new, s.v_new, s.starts, q=s.q if case["rot"] else None, q_out=s.q_out,
                                      rotary=s.rotary)
        else:
            _append_plain(s, s.q_out)
        return s.q_out, c.k, c.v
    if kind == "chunk":
        if own:
            dad.paged_attention_bf16(s.out, s.q, c, s.starts, case["new"], s.scale, lse=s.lse)
        else:
            _chunk_plain(s)
        return s.out, s.lse
    if own:
        dad.decode_attention_paged_bf16(s.out, s.q, s.k_new, s.v_new, c, s.scale, rotary=s.rotary)
    else:
        _decode_plain(s)
    return s.out, c.k, c.v


def work(case):
    """Bytes and FLOPs of one pass: every input read once, every output written once."""
    H, Hkv, D, size = case["H"], case["Hkv"], case["D"], TYPES[case["dtype"]].itemsize
    if case["kind"] == "rotary":
        n = case["B"] * case["S"] * (H + Hkv)
        return {"bytes": 4 * n * D * size, "flops": 2 * n * 3 * case["rot"]}
    ahead, counts = _sizes(case)
    rows, tokens = sum(ahead) + sum(counts), sum(counts)
    pairs = sum(n * a + n * (n + 1) / 2 for a, n in zip(ahead, counts))
    if case["kind"] == "append":
        moved = (2 * Hkv + (H if case["rot"] else 0)) * D
        return {"bytes": tokens * moved * (size + 2), "flops": tokens * (H + Hkv) * 3 * case["rot"]}
    new = 4 * tokens * (H + Hkv) * D if case["kind"] == "decode" else 4 * tokens * H * (D + 1)
    return {"bytes": 4 * Hkv * D * rows + new, "flops": 4 * H * D * pairs}


# ---- in 64 bits -------------------------------------------------------------------------------------------------

def _angles64(case, positions):
    """cos and sin of every (position, pair), from the definition."""
    rot, how = case["rot"], SCALINGS[case["scaling"]]
    cos, sin = [], []
    p = torch.as_tensor(positions, dtype=torch.float64, device="cuda")
    for i in range(rot // 2):
        base, factor = 10000.0, 1.0
        if case["scaling"] == "base":
            base = 10000.0 * how["stretch"] ** (rot / max(rot - 2, 1))
        w = 1.0 / base ** (2 * i / rot)
        if case["scaling"] == "linear":
            w /= how["stretch"]
        if case["scaling"] == "parts":
            r = how["trained_len"] * w / (2 * math.pi)
            gamma = min(1.0, max(0.0, (r - how["low"]) / (how["high"] - how["low"])))
            w = (1 - gamma) * w / how["stretch"] + gamma * w
            factor = 0.1 * math.log(how["stretch"]) + 1
        cos.append(torch.cos(p * w) * factor)
        sin.append(torch.sin(p * w) * factor)
    return torch.stack(cos, -1), torch.stack(sin, -1)


def _turn64(x, case, positions, sign=1):
    """x [n, heads, D] of n positions."""
    cos, sin = _angles64(case, positions)
    cos, sin = cos[:, None], sign * sin[:, None]
    rot = case["rot"]
    y = x.double().clone()
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., first].double(), x[..., second].double()
    y[..., first] = cos * a - sin * b
    y[..., second] = sin * a + cos * b
    return y


def _rows64(s, pool, b, n):
    page = s.case["page"]
    got = torch.empty(pool.shape[1], n, pool.shape[3], dtype=torch.float64, device="cuda")
    for i, p in enumerate(s.cache.page_table[b].tolist()):
        if i * page >= n:
            break
        m = min(page, n - i * page)
        got[:, i * page:i * page + m] = pool[p, :, :m].double()
    return got


def _attend64(q, k, v, first, scale):
    """q [n, H, D] at rows first .. of k, v [Hkv, rows, D] -> out [n, H, D], lse [n, H]."""
    n, H, D = q.shape
    out = torch.empty(n, H, D, dtype=torch.float64, device="cuda")
    lse = torch.empty(n, H, dtype=torch.float64, device="cuda")
    at = first + torch.arange(n, device="cuda")
    late = torch.arange(k.shape[1], device="cuda")[None, :] > at[:, None]
    for h in range(H):
        kv = h // (H // k.shape[0])
        x = torch.einsum("id,jd->ij", q[:, h].double(), k[kv]) * scale
        x[late] = float("-inf")
        top = x.max(1, keepdim=True).values
        e = torch.exp(x - top)
        total = e.sum(1, keepdim=True)
        out[:, h] = torch.einsum("ij,jd->id", e, v[kv]) / total
        lse[:, h] = (top + total.log())[:, 0]
    return out, lse


def exact(case, seed):
    """What run returns, in 64 bits; bytes that are only moved have no other value than their own."""
    if case["kind"] == "append" and not case["rot"]:
        return None
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        at = range(case["first"], case["first"] + case["S"])

        def each(x, sign):
            return torch.stack([_turn64(x[b], case, at, sign) for b in range(case["B"])])

        return each(s.q, 1), each(s.k, 1), each(s.dq_turned, -1), each(s.dk_turned, -1)
    c, page = s.cache, case["page"]
    tables = c.page_table.tolist()
    k_pool = c.k.double() if case["kind"] != "chunk" and case["rot"] else None
    outs, at = [], 0
    for b, (ahead, n) in enumerate(zip(s.ahead, s.counts)):
        rows = range(ahead, ahead + n)
        q = s.q[at:at + n]
        if case["kind"] != "chunk":
            k, v = s.k_new[at:at + n], s.v_new[at:at + n]
            if case["rot"]:
                q, k = _turn64(q, case, rows), _turn64(k, case, rows)
                place = torch.tensor([tables[b][j // page] for j in rows], device="cuda")
                k_pool[place, :, torch.tensor([j % page for j in rows], device="cuda")] = k
        if case["kind"] == "append":
            outs.append((q, None))
        elif case["kind"] == "chunk":
            outs.append(_attend64(q, _rows64(s, c.k, b, ahead + n), _rows64(s, c.v, b, ahead + n), ahead, s.scale))
        else:
            keys, values = (torch.cat((_rows64(s, pool, b, ahead), x.double().transpose(0, 1)), 1)
                            for pool, x in ((c.k, k), (c.v, v)))
            outs.append(_attend64(q, keys, values, ahead, s.scale))
        at += n
    first = torch.cat([x for x, _ in outs])
    if case["kind"] == "append":
        return first, k_pool, None
    if case["kind"] == "chunk":
        return first, torch.cat([x for _, x in outs])
    return first, k_pool, None
