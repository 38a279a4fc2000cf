"""Windowed causal attention and its gradients in float64, with elementwise bounds for bf16 kernels."""
import torch

HALF_BF16 = 2.0 ** -8   # half a step of bf16, relative
U = 2.0 ** -24          # of fp32


def visible(S, window, sinks, device="cpu"):
    i, j = torch.arange(S, device=device)[:, None], torch.arange(S, device=device)[None]
    seen = j <= i
    return seen & ((i - j < window) | (j < sinks)) if window else seen


def forward(q, k, v, scale, window, sinks):
    """[S,D] of one unit -> out, lse, P (float64)."""
    s = (q.double() @ k.double().T) * scale
    s = s.masked_fill(~visible(len(q), window, sinks, q.device), float("-inf"))
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - lse[:, None])
    return p @ v.double(), lse, p


def backward(q, k, v, dout, scale, window, sinks):
    out, _, p = forward(q, k, v, scale, window, sinks)
    do = dout.double()
    ds = p * (do @ v.double().T - (do * out).sum(1, keepdim=True)) * scale
    return ds @ k.double(), ds.T @ q.double(), p.T @ do


def bounds(q, k, v, dout, scale, window, sinks):
    """How far out, lse, dq, dk and dv of a kernel may be off, element by element: it works in fp32 on bf16 operands, rounds
    P and dS to bf16 ahead of the products they go into, forms delta from the rounded out, and rounds results to bf16.
    A score, a sum of D products and a multiplication (D + 4 roundings of the sum of their sizes), moves a probability by
    at most `rel` of itself; ex2, sums of S terms and lse's own rounding are in it, too. (In `reach` also pairs that are
    hidden inside a visited tile contribute exact zeros.)"""
    S, D = q.shape
    q, k, v, do = (t.double() for t in (q, k, v, dout))
    out, lse, p = forward(q, k, v, scale, window, sinks)
    size = (q.abs() @ k.abs().T * scale).masked_fill(~visible(S, window, sinks, q.device), 0.0).amax(1, keepdim=True)
    rel = 2 * (D + 4) * U * size + 2 * (S + 4) * U + 4 * U * lse.abs()[:, None] + 2.0 ** -20   # [S,1]
    h = HALF_BF16
    p_off = p * (rel + h * (1 + rel))                       # as an operand
    e_out = p_off @ v.abs()
    e_out = e_out + h * (out.abs() + e_out)
    dp = do @ v.T
    dp_off = (D + 2) * U * (do.abs() @ v.abs().T)
    delta = (do * out).sum(1, keepdim=True)
    delta_off = (do.abs() * e_out).sum(1, keepdim=True) + (D + 2) * U * (do.abs() * out.abs()).sum(1, keepdim=True)
    ds = p * (dp - delta) * scale
    ds_off = p * (rel + 4 * U) * (dp - delta).abs() * scale + p * (1 + rel) * (dp_off + delta_off) * scale
    ds_off = ds_off + h * (ds.abs() + ds_off)
    sums = (S + 2) * U
    e = [ds_off @ k.abs() + sums * (ds.abs() @ k.abs()), ds_off.T @ q.abs() + sums * (ds.abs().T @ q.abs()),
         p_off.T @ do.abs() + sums * (p.T @ do.abs())]
    grads = (ds @ k, ds.T @ q, p.T @ do)
    e = [x + h * (g.abs() + x) for x, g in zip(e, grads)]
    return e_out, rel[:, 0] + U * lse.abs(), *e
