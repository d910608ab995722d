"""A process's first operator call inside a stream capture: each in a process of its own."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

CHILD = """
import importlib, sys
import torch
sys.path.insert(0, %r)
ops = importlib.import_module("maxim-rs_b200.ops")
g = torch.Generator(device="cuda")
g.manual_seed(1)
x, w = torch.randn(40, 64, generator=g, device="cuda"), torch.randn(48, 64, generator=g, device="cuda")
one = torch.ones(64, device="cuda")
zero = torch.zeros(64, device="cuda")
dy = torch.randn(40, 48, generator=g, device="cuda")
call = {"layer_norm": lambda: ops.layer_norm(x, one, zero), "dense": lambda: ops.dense(x, w, act="gelu"),
        "dense_backward": lambda: ops.dense_backward(dy, x, w)[1]}[sys.argv[1]]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = call()
got.zero_()
graph.replay()
torch.cuda.synchronize()
assert torch.equal(got, call()), "the graph's result differs"
print("fine")
"""


@pytest.mark.parametrize("entry", ["layer_norm", "dense", "dense_backward"])
def test_first_call_in_a_capture(entry):
    r = subprocess.run([sys.executable, "-c", CHILD % ROOT, entry], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr
