"""The paged calls' own scratch: a program that makes none of them does not hold it, and the first of them allocates it, also where
that call is captured into a graph. In a fresh process, since any earlier paged call has made it."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

from gpu_util import need_gpu, say

pytestmark = pytest.mark.gpu

CHILD = r"""
import ctypes as C, sys
import torch
from moa_amd import _lib, ops
lib = _lib.load()

def state():
    v = C.c_uint32(0)
    assert lib.moa_test_scratch_state(C.byref(v)) == 0
    return v.value

def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")

ops.init(0)
assert state() == 3, state()
g = torch.Generator(device="cuda").manual_seed(1)
rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)
k, v = rand(1, 80, 16, 2, 128), rand(1, 80, 16, 2, 128)
cache = ops.PagedCache(k, v, i32([list(range(60)), list(range(60, 80)) + [0] * 40]), i32([900, 300]), i32([1] * 80))
q, starts = rand(42, 8, 128), [i32([0, 40, 42]), i32([0, 1, 2])]
outs, want = [torch.zeros_like(q) for _ in range(2)], [torch.zeros_like(q) for _ in range(2)]
torch.cuda.synchronize()
assert state() == 3, state()

def step(outs):
    ops.paged_attention(q, cache, starts[0], outs[0], max_rows=40)
    ops.paged_attention(q, cache, starts[1], outs[1], max_rows=1)

mode = sys.argv[1]
if mode == "eager":
    step(want)
    assert state() == 7, state()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, capture_error_mode=mode if mode != "eager" else "global"):
    step(outs)
assert state() == 7, state()
for _ in range(3):
    for o in outs:
        o.zero_()
    graph.replay()
    torch.cuda.synchronize()
    step(want)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want)) and all(o.any() for o in outs)
assert ops.device_errors() == 0
print("DONE")
"""


@pytest.mark.parametrize("mode", ["eager", "global", "relaxed"])
def test_the_first_paged_call_makes_the_scratch(mode):
    need_gpu()
    say(f"first paged call of a process, capture mode {mode}")
    root = Path(__file__).resolve().parent.parent
    env = dict(os.environ, PYTHONPATH=os.pathsep.join(str(p) for p in (root / "moa-workspace_amd", root / "tests")))
    res = subprocess.run([sys.executable, "-c", CHILD, mode], capture_output=True, text=True, timeout=100, env=env)
    assert res.returncode == 0 and res.stdout.strip().endswith("DONE"), res.stdout + res.stderr[-3000:]
