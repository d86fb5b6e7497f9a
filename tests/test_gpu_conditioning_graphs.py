"""Captured conditioning calls: the first of a process, and graphs that run at
once (B200 only)."""
import os
import subprocess
import sys

import pytest

import test_gpu_conditioning as base

pytestmark = pytest.mark.gpu

FIRST = """
import sys
sys.path[:0] = {paths!r}
import torch
import test_gpu_conditioning as base
rt = base._rt()
sts = [base._layer_state(100), base._layer_state(101, B=3, S=20, N=400, H=8, Hk=2), base._layer_state(102, B=1, S=40, N=100)]
q, k, v, _ = base._inputs(4, 1, 40, 8, 2, 103)
pk, pv = base._inputs(1, 900, 1, 2, 2, 104)[0][0], base._inputs(1, 900, 1, 2, 2, 105)[0][0]
out = torch.empty_like(q)

def calls():
    for st in sts:
        base._layer(st, rt)
    rt.prefix_attn_fwd(q=q, prefix_k=pk, prefix_v=pv, k=k, v=v, out=out, scale=base.SCALE)

g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    calls()
g.replay()
torch.cuda.synchronize()
got = [st[n].clone() for st in sts for n in base.RESULTS] + [out.clone()]
calls()
torch.cuda.synchronize()
rt.device_status()
want = [st[n] for st in sts for n in base.RESULTS] + [out]
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("same")
"""


def test_the_first_calls_of_a_process_may_be_captured(gpu):
    here = os.path.dirname(os.path.abspath(__file__))
    root = os.path.dirname(here)
    paths = [here, root, os.path.join(root, "minimax-h3-swift_b200")]
    p = subprocess.run([sys.executable, "-c", FIRST.format(paths=paths)], capture_output=True, text=True, timeout=120,
                       cwd=root)
    assert p.returncode == 0 and p.stdout.strip() == "same", p.stderr[-2000:]


def test_two_graphs_replayed_at_once(gpu):
    import torch

    rt = base._rt()
    kw = [dict(seed=106, S=1500, N=600), dict(seed=107, B=3, S=30, N=2000, H=8, Hk=2)]
    sts, want = [base._layer_state(**x) for x in kw], [base._layer_state(**x) for x in kw]
    graphs = [torch.cuda.CUDAGraph() for _ in sts]
    for st, w, g in zip(sts, want, graphs):
        base._layer(w, rt)
        with torch.cuda.graph(g):
            base._layer(st, rt)
    streams = [torch.cuda.Stream() for _ in sts]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for st, w in zip(sts, want):
        assert all(torch.equal(st[n], w[n]) for n in base.RESULTS)
