"""Row operators whose first call in the process is captured into a graph."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash1017-engine_b200")
PROGRAM = """
import sys
import torch
sys.path.insert(0, sys.argv[1])
import ffn_b200 as F
T, H, I, E, K = 300, 256, 128, 16, 4
g = torch.Generator(device="cuda").manual_seed(1)
r = lambda *s: torch.randn(*s, device="cuda", generator=g)
codes = lambda *s: torch.randint(-127, 128, s, device="cuda", generator=g, dtype=torch.int8)
x, w, gate = r(T, H).to(torch.bfloat16), 1 + 0.1 * r(H), torch.sigmoid(r(T, 1))
gu, dn, one = codes(E, 2 * I, H), codes(E, H, I), codes(512, H)
gs, ds, os_ = 0.001 + 0 * r(E, 2 * I), 0.001 + 0 * r(E, H), 0.001 + 0 * r(512)
wide, wx = codes(128, 8192), codes(16, 8192)
wsc, xsc = 0.001 + 0 * r(128), 0.01 + 0 * r(16)
idx = torch.randint(0, E, (T, K), device="cuda", generator=g, dtype=torch.int32)
wt = torch.rand(T, K, device="cuda", generator=g)

def run():
    norm = F.BlockNorm(w, w)
    h, xn, q, s = norm.forward(x, x, gate=gate, codes=True)
    y = F.Int8Experts(F.Int8Matrix(gu, gs), F.Int8Matrix(dn, ds)).forward((q, s), idx, wt, residual=x)
    grads = norm.backward(y, h, dh=x, dxn=x, gate=gate)
    off, pos, src = F.moe_sort(idx, 2, 9)
    xs = F.moe_permute(x, pos, out=torch.zeros(T * K, H, device="cuda", dtype=x.dtype))
    dy, dw = F.moe_combine_backward(x, xs, pos, wt)
    m = F.Int8Matrix(one, os_)
    return [h, y, off, pos, src, xs, dy, dw, m.matmul(x[:1]), m.matmul(x), F.Int8Matrix(wide, wsc).matmul((wx, xsc)),
            *(v for v in grads.values() if v is not None)]

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = run()
graph.replay()
torch.cuda.synchronize()
want = run()
assert all(torch.equal(a, b) for a, b in zip(out, want))
assert all(torch.isfinite(t.float()).all() for t in want)
print("captured")
"""


def test_first_calls_in_a_captured_graph(ffn, cuda):
    r = subprocess.run([sys.executable, "-c", PROGRAM, PKG], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-3000:]
