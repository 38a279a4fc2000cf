"""CPU: the bounds for rows that see few keys hold for the arithmetic that the backward uses, and not for what they are there
to find."""
import pytest
import torch

from tests.window_few_keys import bounds, inputs, rows, worst
from tests.window_reference import visible


def _model(q, k, v, dout, scale, window, sinks, form):
    """The backward's arithmetic in fp32, dS and the results rounded to bf16; delta of the few-key rows by `form`."""
    S = len(q)
    n = rows(S, window, sinks)
    q, k, v, do = (t.float() for t in (q, k, v, dout))
    seen = visible(S, window, sinks)
    s = (q @ k.T * scale).masked_fill(~seen, float("-inf"))
    p = torch.exp(s - torch.logsumexp(s, 1)[:, None])
    dp = do @ v.T
    of_out = (do * (p.bfloat16().float() @ v).bfloat16().float()).sum(1)
    of_pairs = (p * dp).sum(1)
    if form == "a tile lost":   # of eight keys, the last of each row
        at = torch.arange(S)
        of_pairs = (p * dp * (at[None] // 8 < at[:, None] // 8)).sum(1)
    delta = torch.cat([of_out[:n] if form == "of out" else of_pairs[:n], of_out[n:]])
    ds = (p * (dp - delta[:, None])).bfloat16().float()
    return (ds @ k * scale).bfloat16(), (ds.T @ q * scale).bfloat16()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,window,sinks", [(20, 5, 0), (32, 100, 0), (56, 68, 4), (100, 16, 4), (200, 28, 4), (300, 256, 4), (40, 2, 60)])
def test_what_the_bounds_allow(S, window, sinks, D):
    g = torch.Generator().manual_seed(S + D)
    x = [t[0] for t in inputs(1, S, D, g)]
    dq, dk = bounds(*x, D ** -0.5, window, sinks)
    for form, good in (("of pairs", True), ("of out", False), ("a tile lost", False)):
        got = _model(*x, D ** -0.5, window, sinks, form)
        assert (worst(got[0], dq) <= 1.0) == good, form
        if dk is not None and good:
            assert worst(got[1], dk) <= 1.0


def test_which_rows():
    assert [rows(*a) for a in ((32, 0, 0), (33, 0, 0), (500, 28, 4), (500, 28, 5), (500, 1, 31), (20, 400, 400))] == [32, 32, 500, 32, 500, 20]
