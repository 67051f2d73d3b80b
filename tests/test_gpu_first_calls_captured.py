"""A process whose first use of the operators beside the block is inside a graph capture: kernels are loaded, sizes asked
for and shared memory opted in to there.  Each case is a process of its own, since a kernel that ran before is no first call."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

_HEAD = """
import sys
sys.path[:0] = ["tests", "."]
import torch
from _ops64 import attention64, bucket_matrix, check
gen = torch.Generator(device="cuda").manual_seed(3)
r = lambda *s: torch.randn(s, generator=gen, device="cuda").to({dtype})
"""

_ATTENTION = _HEAD + """
B, Lq, Lk, H, D, biased = {sizes}
q, k, v, g = r(B, Lq, H, D), r(B, Lk, H // 2, D), r(B, Lk, H // 2, D), r(B, Lq, H, D)
b = r(1, H, Lq, Lk) if biased else None
m = torch.rand(B, Lk, generator=gen, device="cuda") > 0.3
torch.cuda.synchronize()
from miniworld_engine_b200 import cross_attention_backward_b200, cross_attention_forward_b200
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out, state = cross_attention_forward_b200(q, k, v, bias=b, key_mask=m)
    grads = cross_attention_backward_b200(g, q, k, v, out, state, bias=b, key_mask=m)
for step in range(2):          # new inputs in the same places
    for t in (q, k, v, g):
        t.copy_(r(*t.shape))
    graph.replay()
    torch.cuda.synchronize()
    want = attention64(q, k, v, b, m, None, g)
    for name, t in zip(("out", "dq", "dk", "dv", "dbias"), (out, *grads)):
        if t is not None:
            check(t, want[name], name)
print("right")
"""

_BIAS = _HEAD + """
layout, channels = {sizes}
table, pos = r(33, channels).float(), torch.arange(150, device="cuda")
seg = (pos > 90).int()
u = bucket_matrix(pos, pos, "log", 32, 128, seg, seg).cuda()
shape = (150, 150, channels) if layout == "pair" else (channels, 150, 150)
whole = lambda: torch.randint(-3, 4, shape, generator=gen, device="cuda").to({dtype})
g = whole()
torch.cuda.synchronize()
from miniworld_engine_b200 import PositionBuckets, relative_position_bias_b200, relative_position_bias_backward_b200
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    buckets = PositionBuckets.logarithmic(32, 128, segments=True)
    out = relative_position_bias_b200(table, buckets, pos, q_segment=seg, layout=layout, dtype={dtype})
    grad = relative_position_bias_backward_b200(g, buckets, pos, q_segment=seg, layout=layout)
for step in range(2):
    table.copy_(r(*table.shape))
    g.copy_(whole())
    graph.replay()
    torch.cuda.synchronize()
    want = table[u].to({dtype})
    assert torch.equal(out, want if layout == "pair" else want.movedim(-1, 0))
    flat = (g if layout == "pair" else g.movedim(0, -1)).reshape(-1, channels).double()
    assert torch.equal(grad.double(), torch.zeros(33, channels, dtype=torch.float64, device="cuda").index_add_(0, u.flatten(), flat))
print("right")
"""


@pytest.mark.parametrize("text,sizes,dtype", [
    (_ATTENTION, (2, 77, 300, 4, 64, True), "torch.bfloat16"),
    (_ATTENTION, (1, 40, 4100, 4, 128, False), "torch.bfloat16"),
    (_ATTENTION, (2, 1, 3000, 4, 64, False), "torch.bfloat16"),
    (_ATTENTION, (2, 60, 500, 4, 32, True), "torch.float32"),
    (_BIAS, ("heads", 8), "torch.bfloat16"),
    (_BIAS, ("pair", 64), "torch.float32"),
], ids=["narrow heads", "wide heads, split", "one token", "fp32", "bias of heads", "bias of pairs"])
def test_first_calls_inside_a_capture(text, sizes, dtype):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    got = subprocess.run([sys.executable, "-c", text.format(sizes=sizes, dtype=dtype)], capture_output=True, text=True, cwd=root,
                         timeout=300)
    assert got.returncode == 0 and got.stdout.strip() == "right", got.stderr[-3000:]
