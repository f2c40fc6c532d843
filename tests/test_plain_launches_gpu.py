"""B200CP_PDL=0 makes every launch a plain one: a captured call then holds no dependent launch."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SCRIPT = """
import ctypes as C, torch, paralleltnnlayers_b200 as P
cu = C.CDLL("libcuda.so.1")
n = lambda *s, d=torch.bfloat16: torch.randn(*s, device="cuda").to(d)

def programmatic(call):
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
        call()
    handle, count = C.c_void_p(graph.raw_cuda_graph()), C.c_size_t(0)
    assert cu.cuGraphGetEdges_v2(handle, None, None, None, C.byref(count)) == 0
    a, b, data = (C.c_void_p * count.value)(), (C.c_void_p * count.value)(), (C.c_ubyte * (8 * count.value))()
    assert cu.cuGraphGetEdges_v2(handle, a, b, data, C.byref(count)) == 0
    return sum(data[8 * k + 2] == 1 for k in range(count.value))

x, y, A, B, V = n(400, 64), n(400, 48), n(3, 64, 8), n(3, 8, 48), n(400, 8)
which = torch.randint(3, (400,), device="cuda", dtype=torch.int32)
plan = P.adapter_plan(which, 3)
Wg, Wu = n(64, 256), n(64, 256)
counts = [programmatic(f) for f in (lambda: P.dense_adapters(y, x, A, B, which), lambda: P.dense_adapters(y[:40], x[:40], A, B, which[:40]),
                                    lambda: P.dense_adapters_backward(y, x, V, A, B, plan), lambda: P.dense_gated(x[:40], Wg, Wu),
                                    lambda: P.dense_gated(x, Wg, Wu))]
print("edges", *counts)
"""


@pytest.mark.parametrize("value", ["0", "1"])
def test_the_switch_reaches_the_clusters(value):
    run = subprocess.run([sys.executable, "-c", SCRIPT], cwd=ROOT, env={**os.environ, "B200CP_PDL": value}, capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stderr[-2000:]
    counts = [int(c) for c in run.stdout.split("edges")[1].split()]
    assert len(counts) == 5 and all(c == 0 if value == "0" else c > 0 for c in counts), counts
