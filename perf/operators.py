"""The operators around the KV cache and windowed attention, as cases whose speed is followed.

Kinds of case (``kind``):
  fill_fp8       a prompt's K / V heads into an 8-bit cache: blocks of 64 tokens with a scale for each block and head
  decode_fp8     one token for every sequence against such a cache
  window_train   forward + backward of causal attention with a sliding window and a few first tokens that stay visible
  decode_window  one token for every sequence against a bf16 cache, over a window, or with the attention weights added up
  evict          the rows of a bf16 cache that have gathered the most weight, moved together

Activations are i.i.d. normal values: after layer norm and a projection they are close to that. Buffers for results,
workspaces and caches are made once, as a model's arena does.
"""
from __future__ import annotations

import torch

own = False

BLOCK = 64            # tokens of an 8-bit block
LOWEST = -3.0e38


def _case(name, **c):
    return {"name": name, **c} if name else c


def _fill(name, B, H, S, D, max_len, dtype, ragged):
    return _case(name, kind="fill_fp8", B=B, H=H, S=S, D=D, max_len=max_len, dtype=dtype, ragged=ragged)


def _decode_fp8(name, B, H, D, max_len, longest, window=0, sinks=0):
    return _case(name, kind="decode_fp8", B=B, H=H, D=D, max_len=max_len, longest=longest, window=window, sinks=sinks)


def _train(name, BH, S, D, window, sinks):
    return _case(name, kind="window_train", BH=BH, S=S, D=D, window=window, sinks=sinks)


def _decode_window(name, B, H, D, max_len, longest, window, sinks, weights):
    return _case(name, kind="decode_window", B=B, H=H, D=D, max_len=max_len, longest=longest, window=window,
                 sinks=sinks, weights=weights)


def _evict(name, B, H, D, max_len, longest, budget, recent):
    return _case(name, kind="evict", B=B, H=H, D=D, max_len=max_len, longest=longest, budget=budget, recent=recent)


def listed():
    return [
        # one user's prompt of odd length, from the fp32 heads that DadGPT's own prefill leaves behind
        _fill("fill_fp8_prompt", 1, 12, 301, 64, 1024, "f32", False),
        # a padded batch of prompts behind the bf16 forward
        _fill("fill_fp8_batch", 64, 12, 1024, 64, 1280, "bf16", True),
        # DadGPT's own generation loop, one sequence: latency is what counts
        _decode_fp8("decode_fp8_one", 1, 12, 64, 1024, 700),
        # serving, 64 sequences of mixed length
        _decode_fp8("decode_fp8_64seq", 64, 12, 64, 1280, 1024),
        # a few long conversations on a larger model
        _decode_fp8("decode_fp8_4seq_long", 4, 24, 128, 8192, 8000),
        # fine-tuning on a last, shorter batch of a corpus with a narrow window
        _train("window_train_ragged", 72, 777, 64, 128, 4),
        # GPT-2 124M, batch 16, at full context
        _train("window_train_gpt2_b16", 192, 1024, 64, 256, 4),
        # long context, head size 128, one sequence of 24 heads
        _train("window_train_long", 24, 8192, 128, 1024, 4),
        # serving with the window that the model was trained with
        _decode_window("decode_window_64seq", 64, 12, 64, 1280, 1024, 256, 4, False),
        # serving with a budget: the weights by which rows are let go are gathered as it goes
        _decode_window("decode_weights_64seq", 64, 12, 64, 1280, 1024, 0, 0, True),
        # and the moment when the budget is enforced
        _evict("evict_64seq", 64, 12, 64, 1280, 1024, 512, 64),
        # the same for a few long conversations
        _evict("evict_4seq_long", 4, 24, 128, 8192, 8000, 2048, 256),
    ]


def _log_int(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    kind = rng.choice(["fill_fp8", "decode_fp8", "decode_fp8", "window_train", "window_train", "decode_window",
                       "decode_window", "evict"])
    D = rng.choice([64, 128])
    H = rng.randint(4, 24)
    if kind == "window_train":
        S = _log_int(rng, 32, 8192)
        BH = H * _log_int(rng, 1, 16)
        while BH * S * S > 24 * 8192 * 8192 // (D // 64):
            BH, S = max(1, BH // 2), (S if BH > 1 else S * 2 // 3)
        window = _log_int(rng, 16, 2048)
        return _train(None, BH, S, D, window, rng.choice([0, 1, 4, 4, 16, rng.randint(1, 200)]))
    B = _log_int(rng, 1, 128)
    max_len = _log_int(rng, 128, 8192)
    while B * H * max_len * D > 1e8:   # as in the listed cases
        max_len = max(128, max_len // 2)
        B = max(1, B // 2)
    longest = rng.randint(max_len // 2, max_len - 1)
    if kind == "fill_fp8":
        return _fill(None, B, H, longest, D, max_len, rng.choice(["f32", "bf16"]), rng.random() < 0.7)
    window, sinks = rng.choice([(0, 0), (_log_int(rng, 16, 2048), rng.choice([0, 1, 4, rng.randint(1, 200)]))])
    if kind == "decode_fp8":
        return _decode_fp8(None, B, H, D, max_len, longest, window, sinks)
    if kind == "decode_window":
        return _decode_window(None, B, H, D, max_len, longest, window, sinks, rng.random() < 0.5)
    budget = rng.randint(max_len // 8, max_len // 2)
    return _evict(None, B, H, D, max_len, longest, budget, rng.randint(0, budget))


class _State:
    pass


def _lengths(g, B, longest):
    """One length in each of B equal parts of 1..longest, in random order."""
    part = torch.rand(B, generator=g, device="cuda") + torch.arange(B, device="cuda")
    part = part[torch.randperm(B, generator=g, device="cuda")]
    return (1 + part * (longest / B)).to(torch.int32).clamp_(max=longest)


def _values(g, dtype, *shape):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, 1.0, generator=g)


class _Cache:
    """What the caches below have in common with the framework's: tensors and sizes."""

    def __init__(self, B, H, max_len, D, fp8, weights):
        self.B, self.H, self.max_len, self.D = B, H, max_len, D
        kind = torch.float8_e4m3fn if fp8 else torch.bfloat16
        self.k = torch.zeros(B, H, max_len, D, device="cuda").to(kind)
        self.v = torch.zeros(B, H, max_len, D, device="cuda").to(kind)
        if fp8:
            self.k_scale = torch.ones(B, H, max(1, max_len // BLOCK), device="cuda")
            self.v_scale = torch.ones_like(self.k_scale)
            self.k_tail = torch.zeros(B, H, BLOCK, D, dtype=torch.bfloat16, device="cuda")
            self.v_tail = torch.zeros_like(self.k_tail)
        self.weights = torch.zeros(B, H, max_len, device="cuda") if weights else None
        self.lengths = torch.zeros(B, dtype=torch.int32, device="cuda")


def _cache(B, H, max_len, D, fp8=False, weights=False):
    if own:   # the framework's cache has a workspace of its own beside the same tensors
        import dadgpt_b200 as dad
        return dad.KVCacheFP8(B, H, max_len, D) if fp8 else dad.KVCacheBF16(B, H, max_len, D, weights=weights)
    return _Cache(B, H, max_len, D, fp8, weights)


def prepare(case, seed):
    s = _State()
    s.case = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, D = case["kind"], case["D"]
    s.scale = D ** -0.5
    if kind == "window_train":
        shape = (case["BH"], case["S"], D)
        s.q, s.k, s.v, s.dout = (_values(g, torch.bfloat16, *shape) * 0.5 for _ in range(4))
        s.out, s.dq, s.dk, s.dv = (torch.empty_like(s.q) for _ in range(4))
        s.lse = torch.empty(shape[:2], device="cuda")
        s.workspace = None
        if own:
            from dadgpt_b200 import attention as dad
            s.workspace = torch.empty(dad.flash_backward_bf16_window_workspace_bytes(*shape), dtype=torch.uint8, device="cuda")
        return s
    B, H, L = case["B"], case["H"], case["max_len"]
    if kind == "fill_fp8":
        s.cache = _cache(B, H, L, D, fp8=True)
        dtype = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
        s.k_heads, s.v_heads = (_values(g, dtype, B, H, case["S"], D) for _ in range(2))
        s.counts = _lengths(g, B, case["S"]) if case["ragged"] else torch.full((B,), case["S"], dtype=torch.int32, device="cuda")
        return s
    s.start = _lengths(g, B, case["longest"])
    k, v = (_values(g, torch.bfloat16, B, H, L, D) for _ in range(2))
    if kind == "evict":
        s.src, s.dst = _cache(B, H, L, D, weights=True), _cache(B, H, L, D, weights=True)
        s.src.k.copy_(k)
        s.src.v.copy_(v)
        s.src.lengths.copy_(s.start)
        # a few rows gather most of the weight
        s.src.weights.exponential_(generator=g).pow_(3.0)
        return s
    fp8 = kind == "decode_fp8"
    s.cache = _cache(B, H, L, D, fp8, case.get("weights", False))
    if fp8:
        _fill_plain(s.cache, k, v, s.start)
    else:
        s.cache.k.copy_(k)
        s.cache.v.copy_(v)
    s.q, s.k_new, s.v_new = (_values(g, torch.bfloat16, B, H, D) for _ in range(3))
    s.out = torch.empty_like(s.q)
    if case.get("weights"):
        s.weights_start = torch.empty(B, H, L, device="cuda").exponential_(generator=g)
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------

def _quantised(x):
    """[..., tokens, D] in whole blocks -> e4m3 values of the same shape, a power of two for each block: the least that
    keeps the block's largest value within 448 = 0.875 * 2^9."""
    blocks = x.float().unflatten(-2, (-1, BLOCK))
    most = blocks.abs().amax((-1, -2))
    mantissa, exponent = torch.frexp(most)
    exponent = torch.where(most > 0, exponent - 9 + (mantissa > 0.875), -126).clamp(min=-126)
    scale = torch.ldexp(torch.ones_like(mantissa), exponent)
    return (blocks / scale[..., None, None]).to(torch.float8_e4m3fn).flatten(-3, -2), scale


def _fill_plain(cache, k_heads, v_heads, counts):
    S = k_heads.shape[2]
    whole = min(S, cache.max_len) // BLOCK
    n = counts.long()
    blocks = torch.arange(whole, device="cuda") < (n // BLOCK)[:, None]            # [B, whole]
    rows = blocks.repeat_interleave(BLOCK, 1)[:, None, :, None]
    open_row = (n // BLOCK * BLOCK)[:, None] + torch.arange(BLOCK, device="cuda")  # [B, BLOCK]
    in_tail = (open_row < n[:, None])[:, None, :, None]
    for data, scales, tail, heads in ((cache.k, cache.k_scale, cache.k_tail, k_heads),
                                      (cache.v, cache.v_scale, cache.v_tail, v_heads)):
        heads = heads.to(torch.bfloat16)
        if whole:
            codes, scale = _quantised(heads[:, :, :whole * BLOCK])
            at = data[:, :, :whole * BLOCK]
            at.copy_(torch.where(rows, codes.float(), at.float()))
            scales[:, :, :whole] = torch.where(blocks[:, None], scale, scales[:, :, :whole])
        take = open_row.clamp(max=S - 1)[:, None, :, None].expand(-1, heads.shape[1], -1, heads.shape[3])
        tail.copy_(torch.where(in_tail, heads.gather(2, take), tail))
    cache.lengths.copy_(counts)


def _visible(positions, keys, window, sinks):
    seen = keys <= positions
    if window:
        seen &= (positions - keys < window) | (keys < sinks)
    return seen


def _attend(q, k, v, seen, scale):
    """One query for each (sequence, head): [B,H,D], [B,H,L,D], [B,L] -> out, probabilities."""
    scores = (q.float()[:, :, None] * k).sum(-1) * scale
    scores = scores.masked_fill(~seen[:, None], LOWEST)
    p = torch.exp(scores - scores.amax(-1, keepdim=True)) * seen[:, None]
    p = p / p.sum(-1, keepdim=True)
    return (p[..., None] * v).sum(2), p


def _decode_fp8_plain(s):
    c, case = s.cache, s.case
    n = c.lengths.long()
    b = torch.arange(c.B, device="cuda")
    c.k_tail[b, :, n % BLOCK], c.v_tail[b, :, n % BLOCK] = s.k_new, s.v_new
    rows = torch.arange(c.max_len, device="cuda")
    opened = rows[None] >= (n // BLOCK * BLOCK)[:, None]                          # [B, L]: rows held in the tail
    whole = max(1, c.max_len // BLOCK)

    def values(data, scales, tail):
        scale = scales[:, :, (rows // BLOCK).clamp(max=whole - 1)][..., None]
        late = tail.float()[:, :, rows % BLOCK]
        return torch.where(opened[:, None, :, None], late, data.float() * scale)

    seen = _visible(n[:, None], rows[None], case["window"], case["sinks"])
    out, _ = _attend(s.q, values(c.k, c.k_scale, c.k_tail), values(c.v, c.v_scale, c.v_tail), seen, s.scale)
    s.out.copy_(out)
    full = (n + 1) % BLOCK == 0                                                    # a block is complete: to 8 bits
    at = (n // BLOCK).clamp(max=whole - 1)
    block_rows = (at * BLOCK)[:, None] + torch.arange(BLOCK, device="cuda")
    block_rows = block_rows.clamp(max=c.max_len - 1)
    for data, scales, tail in ((c.k, c.k_scale, c.k_tail), (c.v, c.v_scale, c.v_tail)):
        codes, scale = _quantised(tail)
        index = block_rows[:, None, :, None].expand(-1, c.H, -1, c.D)
        bits = data.view(torch.uint8)
        keep = bits.gather(2, index)
        bits.scatter_(2, index, torch.where(full[:, None, None, None], codes.view(torch.uint8), keep))
        old = scales[b, :, at]
        scales[b, :, at] = torch.where(full[:, None], scale[..., 0], old)
    c.lengths.copy_(c.lengths + 1)


def _decode_window_plain(s):
    c, case = s.cache, s.case
    n = c.lengths.long()
    b = torch.arange(c.B, device="cuda")
    c.k[b, :, n], c.v[b, :, n] = s.k_new, s.v_new
    rows = torch.arange(c.max_len, device="cuda")
    seen = _visible(n[:, None], rows[None], case["window"], case["sinks"])
    out, p = _attend(s.q, c.k.float(), c.v.float(), seen, s.scale)
    s.out.copy_(out)
    if case["weights"]:
        new = rows[None] == n[:, None]
        c.weights.copy_(torch.where(new[:, None], p, c.weights + p))
    c.lengths.copy_(c.lengths + 1)


def _evict_plain(s):
    case, src, dst = s.case, s.src, s.dst
    budget, recent, L = case["budget"], case["recent"], case["max_len"]
    n = src.lengths.long()[:, None, None]
    rows = torch.arange(L, device="cuda")
    key = torch.where(rows < n - recent, src.weights, -1.0)                         # weights are not negative
    key = torch.where((rows >= n - recent) & (rows < n), float("inf"), key)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices          # equal ones: lowest index first
    rank = torch.empty_like(order).scatter_(-1, order, rows.expand_as(order))
    kept = (rank < budget) & (rows < n)
    place = torch.where(kept, rows, L)
    place = torch.sort(place, dim=-1).values[..., :budget]                         # kept rows, in order; L behind them
    good = place < L
    place = place.clamp(max=L - 1)
    for to, rows_of in ((dst.k, src.k), (dst.v, src.v)):
        got = rows_of.gather(2, place[..., None].expand(-1, -1, -1, case["D"]))
        to[:, :, :budget] = torch.where(good[..., None], got, to[:, :, :budget])
    dst.weights[..., :budget] = torch.where(good, src.weights.gather(2, place), dst.weights[..., :budget])
    dst.lengths.copy_(src.lengths.clamp(max=budget))


def _train_plain(s):
    case = s.case
    at = torch.arange(case["S"], device="cuda")
    seen = _visible(at[:, None], at[None], case["window"], case["sinks"])
    q, k, v, dout = s.q.float(), s.k.float(), s.v.float(), s.dout.float()
    p = torch.baddbmm(torch.zeros((), device="cuda"), q, k.mT, beta=0, alpha=s.scale).masked_fill_(~seen, float("-inf"))
    s.lse.copy_(torch.logsumexp(p, -1))
    p = p.sub_(s.lse[..., None]).exp_()
    out = p @ v
    s.out.copy_(out)
    s.dv.copy_(p.mT @ dout)
    ds = dout @ v.mT
    ds = ds.sub_((dout * out).sum(-1, keepdim=True)).mul_(p).mul_(s.scale)
    del p
    s.dq.copy_(ds @ k)
    s.dk.copy_(ds.mT @ q)


# ---- one pass ---------------------------------------------------------------------------------------------------

def run(s):
    case = s.case
    kind = case["kind"]
    if own:
        from dadgpt_b200 import attention as dad
    if kind == "fill_fp8":
        c = s.cache
        if own:
            dad.kv_cache_fill_fp8(c, s.k_heads, s.v_heads, s.counts)
        else:
            _fill_plain(c, s.k_heads, s.v_heads, s.counts)
        return c.k, c.v, c.k_scale, c.v_scale, c.k_tail, c.v_tail, c.lengths
    if kind == "window_train":
        if own:
            BH, S, D, window, sinks = (case[x] for x in ("BH", "S", "D", "window", "sinks"))
            dad.gpu_flash_attention_forward_bf16_window(s.out, s.lse, s.q, s.k, s.v, BH, S, D, s.scale, window, sinks)
            dad.gpu_flash_attention_backward_bf16_window(s.dq, s.dk, s.dv, s.workspace, s.dout, s.out, s.lse, s.q, s.k,
                                                         s.v, BH, S, D, s.scale, window, sinks)
        else:
            _train_plain(s)
        return s.out, s.lse, s.dq, s.dk, s.dv
    if kind == "evict":
        if own:
            dad.kv_cache_evict_bf16(s.dst, s.src, case["budget"], case["recent"])
        else:
            _evict_plain(s)
        return s.dst.k, s.dst.v, s.dst.weights, s.dst.lengths
    c = s.cache
    c.lengths.copy_(s.start)   # the same token again
    if kind == "decode_fp8":
        if own:
            dad.decode_attention_fp8(s.out, s.q, s.k_new, s.v_new, c, s.scale, window=case["window"], sinks=case["sinks"])
        else:
            _decode_fp8_plain(s)
        return s.out, c.k, c.v, c.k_scale, c.v_scale, c.k_tail, c.v_tail, c.lengths
    if case["weights"]:
        c.weights.copy_(s.weights_start)
    if own:
        dad.decode_attention_bf16_window(s.out, s.q, s.k_new, s.v_new, c, s.scale, window=case["window"],
                                         sinks=case["sinks"], weights=case["weights"])
    else:
        _decode_window_plain(s)
    return s.out, c.k, c.v, c.lengths, c.weights


def _mean_rows(case):
    """Rows that a token sees, on average over the lengths 1..longest, the appended one among them."""
    most = case["longest"]
    if not case["window"]:
        return 1 + (1 + most) / 2
    return sum(min(n + 1, case["window"] + min(case["sinks"], max(0, n + 1 - case["window"])))
               for n in range(1, most + 1)) / most


def work(case):
    """Bytes and FLOPs of one pass: every input read once, every output written once."""
    kind, D = case["kind"], case["D"]
    if kind == "window_train":
        BH, S, W, sinks = case["BH"], case["S"], case["window"], case["sinks"]
        pairs = BH * sum(min(i + 1, W + min(sinks, max(0, i + 1 - W))) for i in range(S))
        return {"bytes": 8 * BH * S * D * 2 + 4 * BH * S, "flops": 14 * D * pairs}
    B, H = case["B"], case["H"]
    if kind == "fill_fp8":
        rows = B * (1 + case["S"]) / 2 if case["ragged"] else B * case["S"]
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": 2 * H * D * rows * (size + 1) + 8 * H * rows / BLOCK, "flops": 4 * H * D * rows}
    if kind == "evict":
        most, budget = case["longest"], case["budget"]
        kept = B * sum(min(n, budget) for n in range(1, most + 1)) / most
        rows = B * (1 + most) / 2
        return {"bytes": H * (kept * (2 * 2 * D * 2 + 4) + rows * 4), "flops": H * rows}
    rows = B * _mean_rows(case)
    token = 6 * B * H * D * 2
    if kind == "decode_fp8":   # on average half a block is in bf16
        late = B * min(BLOCK / 2, rows / B)
        return {"bytes": 2 * H * D * (rows + late) + 8 * H * rows / BLOCK + token, "flops": 4 * H * D * rows}
    return {"bytes": 4 * H * D * rows + (8 * H * rows if case["weights"] else 0) + token, "flops": 4 * H * D * rows}


# ---- in 64 bits -------------------------------------------------------------------------------------------------

def _softmax64(scores):
    e = torch.exp(scores - scores.max())
    return e / e.sum()


def _rows64(case, length):
    """The rows that the token at `length` sees."""
    W = case["window"] or length + 1
    first = max(0, length + 1 - W)
    return list(range(min(case["sinks"], first))) + list(range(first, length + 1))


def _exact_train(s, case):
    S, W, sinks = case["S"], case["window"], case["sinks"]
    i = torch.arange(S, device="cuda").unsqueeze(1)
    j = torch.arange(S, device="cuda").unsqueeze(0)
    hidden = (j > i) | ((j <= i - W) & (j >= sinks))
    got = [[], [], [], [], []]
    for u in range(case["BH"]):
        q, k, v, do = (t[u].double() for t in (s.q, s.k, s.v, s.dout))
        scores = torch.einsum("id,jd->ij", q, k) / case["D"] ** 0.5
        scores[hidden] = float("-inf")
        top = scores.max(1, keepdim=True).values
        weight = torch.exp(scores - top)
        total = weight.sum(1, keepdim=True)
        prob = weight / total
        out = torch.einsum("ij,jd->id", prob, v)
        dprob = torch.einsum("id,jd->ij", do, v)
        dscore = prob * (dprob - (prob * dprob).sum(1, keepdim=True)) / case["D"] ** 0.5
        for to, x in zip(got, (out, (top + total.log())[:, 0], torch.einsum("ij,jd->id", dscore, k),
                               torch.einsum("ij,id->jd", dscore, q), torch.einsum("ij,id->jd", prob, do))):
            to.append(x)
    return tuple(torch.stack(x) for x in got)


def _exact_decode(s, case):
    B, H, D = case["B"], case["H"], case["D"]
    fp8 = case["kind"] == "decode_fp8"
    out = torch.empty(B, H, D, dtype=torch.float64, device="cuda")
    weights = s.weights_start.double() if case.get("weights") else None
    for b, n in enumerate(s.start.tolist()):
        sides = []
        for data, new in ((s.cache.k, s.k_new), (s.cache.v, s.v_new)):
            rows = data[b, :, :n].double()
            if fp8:
                scales, tail = (s.cache.k_scale, s.cache.k_tail) if data is s.cache.k else (s.cache.v_scale, s.cache.v_tail)
                done = n // BLOCK * BLOCK
                steps = scales[b, :, :n // BLOCK].double().repeat_interleave(BLOCK, 1)
                rows = torch.cat([rows[:, :done] * steps[..., None], tail[b, :, :n - done].double()], 1)
            sides.append(torch.cat([rows, new[b].double()[:, None]], 1))
        at = torch.tensor(_rows64(case, n), device="cuda")
        k, v = (x[:, at] for x in sides)
        scores = torch.einsum("hd,hjd->hj", s.q[b].double(), k) / D ** 0.5
        prob = torch.exp(scores - scores.max(1, keepdim=True).values)
        prob /= prob.sum(1, keepdim=True)
        out[b] = torch.einsum("hj,hjd->hd", prob, v)
        if weights is not None:
            weights[b, :, n] = 0.0
            weights[b, :, at] += prob
    if fp8:
        return (out,) + (None,) * 7
    return out, None, None, None, weights


def exact(case, seed):
    """What run returns, in 64 bits; bytes that are only moved or rounded have no other value than their own."""
    if case["kind"] in ("fill_fp8", "evict"):
        return None
    s = prepare(case, seed)
    return _exact_train(s, case) if case["kind"] == "window_train" else _exact_decode(s, case)
