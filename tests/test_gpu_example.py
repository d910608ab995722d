"""examples/train_mlp.py: the operators together, as a user trains and serves a block with them."""
import importlib.util
import os

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_mlp", os.path.join(ROOT, "examples", "train_mlp.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_the_block_learns_and_serves(example, dtype):
    block, x, losses = example.train(500, 96, 60, example.DTYPES[dtype])
    assert losses[-1] < 0.5 * losses[0], (losses[0], losses[-1])
    whole = block.serve(x[:9])
    # One token goes through other kernels; both round each of three results to the type once.
    unit = {"f32": 2.0 ** -18, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    for i in range(9):
        one = block.serve(x[i:i + 1])
        assert (one.float() - whole[i:i + 1].float()).abs().max() <= 8 * unit * whole[i].float().abs().max()


def test_the_blocks_gradients_match_autograd(example):
    """Against torch's own gradients of the same block in 64 bits. fp32 sums of a
    few hundred terms: 1e-5 of each gradient's size."""
    block = example.Mlp(40, 160, torch.float32, 3)
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    x, dy = (torch.randn(150, 40, generator=g, device="cuda") for _ in range(2))
    y, saved = block.forward(x)
    dx, grads = block.backward(dy, saved)
    p = {k: v.double().requires_grad_() for k, v in block.p.items()}
    xd = x.double().requires_grad_()
    n = torch.nn.functional.layer_norm(xd, (40,), p["scale"], p["shift"], 1e-6)
    h = torch.nn.functional.gelu(n @ p["w1"].t() + p["b1"])
    want = xd + h @ p["w2"].t() + p["b2"]
    want.backward(dy.double())
    assert (y.double() - want).norm() <= 1e-5 * want.norm()
    assert (dx.double() - xd.grad).norm() <= 1e-5 * xd.grad.norm()
    for k, v in grads.items():
        assert (v.double() - p[k].grad).norm() <= 1e-5 * p[k].grad.norm(), k
