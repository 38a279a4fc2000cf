"""GPU: a call on rotary positions or a paged cache that is the first on its device may come while a stream is being captured, its
own or another. Each in a fresh process."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = """
import sys, torch
import dadgpt_b200 as dad
path, where = sys.argv[1:]
B, H, D = 2, 3, 64
c = dad.KVCachePagedBF16(B, H, 40, 16, 20, D)
c.page_table.copy_(torch.arange(40).view(2, 20))
c.lengths.copy_(torch.tensor([100, 7], dtype=torch.int32))
r = dad.RotaryPositions(D)
starts = torch.tensor([0, 30, 31], dtype=torch.int32, device="cuda")
q, k, v = (torch.randn(31, H, D, device="cuda").bfloat16() for _ in range(3))
out, y = torch.zeros_like(q), torch.zeros(4, device="cuda")

def call():
    if path == "rotary":
        dad.rotary_forward(out[None], None, q[None], None, r)
    elif path == "append":
        dad.kv_cache_append_paged(c, k, v, starts, q=q, q_out=out, rotary=r)
    elif path == "attention":
        dad.paged_attention_bf16(out, q, c, starts, 30, 0.125)
    else:
        dad.decode_attention_paged_bf16(out[:B], q[:B], k[:B], v[:B], c, 0.125, rotary=r)

c.v.normal_()
other = torch.cuda.Stream()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, capture_error_mode="global"):
    y.add_(1.0)
    if where == "own":
        call()
    else:
        with torch.cuda.stream(other):
            call()
if where == "own":
    torch.cuda.synchronize()
    assert not out.any()
graph.replay()
torch.cuda.synchronize()
assert y.eq(1.0).all() and out.any() and out.isfinite().all()
assert dad.attention.device_status() == 0
"""


@pytest.mark.parametrize("path,where", [("rotary", "own"), ("append", "own"), ("attention", "own"), ("attention", "other"),
                                        ("decode", "own"), ("decode", "other")])
def test_first_call_during_a_capture(cuda, path, where):
    r = subprocess.run([sys.executable, "-c", SCRIPT, path, where], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
