"""The first call of a process may lie inside a stream capture."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import torch
from piccl_b200.ops import fp8
from piccl_b200.ops.optimizer import AdamW

def layer(M, N, K):
    x, dy, w = torch.randn(M, K, device="cuda").bfloat16(), torch.randn(M, N, device="cuda").bfloat16(), torch.randn(N, K, device="cuda")
    out = torch.empty(M, N, device="cuda", dtype=torch.bfloat16), torch.empty(M, K, device="cuda", dtype=torch.bfloat16), torch.empty(N, K, device="cuda")
    return x, dy, w, fp8.empty(N, K), fp8.empty(K, N), fp8.empty(K, M), out

layers = [layer(300, 264, 520), layer(1, 264, 520), layer(24, 264, 520), layer(1, 5000, 264)]
p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
opts = [AdamW([p], [g], bits=8), AdamW([p], [g])]

def step():
    for x, dy, w, w8, w8t, xt, (y, dx, dw) in layers:
        fp8.quantize(w, w8, transposed=w8t, square=True)
        fp8.linear(x, w8, y)
        fp8.linear(x, w8, y, keep=xt)
        fp8.linear_bwd(dy, xt, w8t, dx, dw)
    for o in opts:
        o.step(1e-3)

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    step()
graph.replay()
got = [[t.clone() for t in l[-1]] for l in layers]
step()
assert all(torch.equal(a, b) for l, q in zip(layers, got) for a, b in zip(l[-1], q))
assert all(int(o.step_dev) == 2 for o in opts)
print("fine")
"""


def test_the_first_calls_of_a_process_are_captured():
    r = subprocess.run([sys.executable, "-c", PROGRAM], capture_output=True, text=True, timeout=300, cwd=Path(__file__).resolve().parent.parent)
    assert r.returncode == 0 and r.stdout.strip().endswith("fine"), r.stderr[-2000:]
