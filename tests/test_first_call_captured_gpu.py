"""The very first calls of a process made while a stream is captured into a graph: nothing that a
first call sets up (kernel attributes, occupancy, code loading) may break the capture, and the
replay gives the eager calls' bits."""
import os
import subprocess
import sys

import pytest

pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = """
import sys
sys.path.insert(0, sys.argv[1])
import torch, qgemm
side = torch.cuda.Stream()
dev = qgemm.Device(0)
st = dev.wrap_stream(side.cuda_stream)
ops = qgemm.QuantizedGemmOps(st)
g = torch.Generator("cuda").manual_seed(1)
def bf(*s):
    return torch.randn(*s, generator=g, device="cuda").bfloat16()
def i8(*s):
    return torch.randint(-127, 128, s, generator=g, device="cuda", dtype=torch.int8)
T, E, k, H = 600, 300, 2, 256
x, w1, wp, w8 = bf(1, 4096), bf(512, 4096), bf(2304, 256), i8(E, H, H)
xp, logits = bf(2048, 256), torch.randn(T, E, generator=g, device="cuda")
xt, sw = bf(T, H), torch.rand(E, H, generator=g, device="cuda") / 2000
o1, op = torch.empty(1, 512, device="cuda"), torch.empty(2048, 2304, device="cuda").bfloat16()
wt, ex = torch.empty(T, k, device="cuda"), torch.empty(T, k, dtype=torch.int32, device="cuda")
off, rows = torch.empty(E + 1, dtype=torch.int32, device="cuda"), torch.empty_like(ex)
q, sq = torch.empty(T * k, H, dtype=torch.int8, device="cuda"), torch.empty(T * k, device="cuda")
h, out = torch.empty(T * k, H, device="cuda").bfloat16(), torch.empty(T, H, device="cuda").bfloat16()
outs = [o1, op, wt, ex, off, rows, q, sq, h, out]
def calls():
    ops.linearBf16NK(x, w1, o1, 1, 512, 4096, out_dtype=qgemm.F32)
    ops.linearBf16NK(xp, wp, op, 2048, 2304, 256)
    ops.routeTopK(logits, wt, ex, off, rows, T, E, k)
    ops.dispatchRowsQuantized(xt, rows, q, sq, T, k, H, T * k)
    ops.w8a8ExpertLinear(q, w8, sq, sw, off, h, E, T * k, H, H)
    ops.combineRows(h, rows, wt, out, T, k, H, T * k)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    calls()
graph.replay()
torch.cuda.synchronize()
st.sync()
kept = [o.clone() for o in outs]
for o in outs:
    o.zero_()
torch.cuda.synchronize()
calls()
st.sync()
for i, (a, b) in enumerate(zip(kept, outs)):
    assert torch.equal(a, b), i
    assert a.float().abs().sum() > 0, i
print("same bits")
"""


def test_first_calls_inside_a_capture():
    r = subprocess.run([sys.executable, "-c", SCRIPT, os.path.join(ROOT, "cuda-triton-scala_b200")],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    assert "same bits" in r.stdout
