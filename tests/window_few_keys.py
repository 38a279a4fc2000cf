"""dQ and dK of rows that see few keys, whose delta the windowed backward forms from P and dP (csrc/window_delta.cuh): the bounds
that hold for these rows only."""
import torch

from tests.window_reference import HALF_BF16, backward, forward, visible

FEW = 32               # kFewKeys
STEP = 2.0 ** -23      # of fp32, relative: a product or sum of the matrix instructions may be cut off rather than rounded


def rows(S, window, sinks):
    """Which rows these are: all of them where no row sees more than FEW keys, else the first FEW."""
    return S if S <= FEW or window and window + sinks <= FEW else FEW


def bounds(q, k, v, dout, scale, window, sinks):
    """[S,D] of one unit -> dq and how far it may be off in the rows above; dk and its bound where these are all rows, else None.
    P comes from a score, a sum of D products scaled (D + 4 steps of the sum of their sizes), and lse, which has the scores' and
    the sums' errors once more: off by `rel` of itself, ex2 among it. delta is a sum of at most 2 FEW products of P and dP. dS is
    rounded to bf16 once, and the results once; there is no O in it."""
    S, D = q.shape
    n = rows(S, window, sinks)
    q, k, v, do = (t.double() for t in (q, k, v, dout))
    _, lse, p = forward(q, k, v, scale, window, sinks)
    hidden = ~visible(S, window, sinks, q.device)
    size = (q.abs() @ k.abs().T * scale).masked_fill(hidden, 0.0).amax(1, keepdim=True)
    rel = 2 * (D + 4) * STEP * size + 2 * (FEW + 4) * STEP + 4 * STEP * lse.abs()[:, None] + 2.0 ** -20
    dp = do @ v.T
    dp_off = (D + 2) * STEP * (do.abs() @ v.abs().T)
    delta = (p * dp).sum(1, keepdim=True)
    delta_off = (p * ((rel + 2 * FEW * STEP) * dp.abs() + (1 + rel) * dp_off)).sum(1, keepdim=True)
    ds = p * (dp - delta) * scale
    ds_off = p * (rel + 4 * STEP) * (dp - delta).abs() * scale + p * (1 + rel) * (dp_off + delta_off) * scale
    ds_off = ds_off + HALF_BF16 * (ds.abs() + ds_off)
    sums = (S + 2) * STEP
    dq, dk, _ = backward(q, k, v, dout, scale, window, sinks)
    off = ds_off @ k.abs() + sums * (ds.abs() @ k.abs())
    dq_off = off + HALF_BF16 * (dq.abs() + off)
    off = ds_off.T @ q.abs() + sums * (ds.abs().T @ q.abs())
    dk_off = off + HALF_BF16 * (dk.abs() + off)
    return (dq[:n], dq_off[:n]), ((dk, dk_off) if n == S else None)


def inputs(BH, S, D, generator, device="cpu"):
    """q, k, v, dout [BH,S,D] bf16. The rows of V have most of themselves in common, so that dP of a row's pairs hardly differ
    and dS is small beside delta: an error of delta shows."""
    q, k, v, do = (torch.randn(BH, S, D, device=device, generator=generator) for _ in range(4))
    common = 4 * torch.randn(BH, 1, D, device=device, generator=generator)
    return [x.bfloat16() for x in (q, k, v + common, do)]


def worst(got, want):
    """The largest error, as a share of what is allowed."""
    value, allowed = want
    return ((got[:len(value)].double() - value).abs() / (allowed + 1e-30)).max().item()
