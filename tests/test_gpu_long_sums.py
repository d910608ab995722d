"""Sums over many rows or a long K, of one sign: where the tensor core's truncating
accumulator would show as a bias.

What a set of accumulators takes before it goes to registers bounds the loss: at
most 256 updates in 16 bits, 32 in fp32, each cutting the sum so far by less than
2^-23 of it. To that fp32 adds its split (the product of the two low halves, at most
2^-20, and both low halves' rounding, 2^-21 each), and every output its own
rounding. Of one set over 131,072 of K the loss was 7.8e-4."""
import importlib
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_ops import DENSE_MKN  # noqa: E402

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
LOSS = {F32: 32 * 2.0 ** -23 + 2.0 ** -20 + 2 * 2.0 ** -21, BF16: 256 * 2.0 ** -23, F16: 256 * 2.0 ** -23}


@pytest.fixture(scope="module")
def ops():
    return importlib.import_module("maxim-rs_b200.ops")


def positive(seed, rows, cols, dtype, spread=False):
    """Uniform over (0, 1/8); `spread` scales the columns by 1 to 2, so that sums fall all over a binade and
    their own roundings average out."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = torch.rand(rows, cols, generator=g, device="cuda") / 8
    if spread:
        t *= torch.exp2(torch.rand(cols, generator=g, device="cuda"))
    return t.to(dtype)


def sums(a, b):
    """a^T b in 64 bits, by pieces."""
    t = torch.zeros(a.shape[1], b.shape[1], dtype=torch.float64, device="cuda")
    for i in range(0, a.shape[0], 8192):
        t.addmm_(a[i:i + 8192].double().t(), b[i:i + 8192].double())
    return t


def check(got, want):
    err = (got.double() - want) / want
    loss, u = LOSS[got.dtype], U[got.dtype]
    assert err.abs().max().item() <= loss + 1.001 * u, (err.abs().max().item(), loss + u)
    # Roundings to nearest average out: over N outputs to u / sqrt(N), six of which are allowed.
    assert abs(err.mean().item()) <= loss + 6 * u / got.numel() ** 0.5, (err.mean().item(), loss)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("mkn", [(131072, 2304, 2304), (131072, 1024, 776), (131072, 136, 256), (131071, 64, 40),
                                 (20000, 2304, 2304)])
def test_weight_gradients_of_one_sign(ops, mkn, dtype):
    m, k, n = mkn
    dy, x = positive(1, m, n, dtype, spread=True), positive(2, m, k, dtype)
    w = torch.empty(n, k, dtype=dtype, device="cuda")
    _, dw, _ = ops.dense_backward(dy, x, w, need_dx=False, need_db=False)
    ops.poll()
    check(dw, sums(dy, x))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("mkn", [(520, 131072, 136), (3000, 20000, 3000), (40, 70001, 64)])
def test_products_of_one_sign(ops, mkn, dtype):
    m, k, n = mkn
    x, w = positive(3, k, m, dtype, spread=True).t().contiguous(), positive(4, k, n, dtype).t().contiguous()
    y = ops.dense(x, w)
    ops.poll()
    check(y, sums(x.t(), w.t()))


@pytest.mark.parametrize("mkn", DENSE_MKN)
def test_fp32_split_at_every_size(ops, mkn):
    """Each of the three products of fp32 operands, where a low half left out or a set that took too much
    would show (tests/test_fp32_bound.py: what fails this bound)."""
    m, k, n = mkn
    x, w, dy = positive(5, m, k, F32), positive(6, n, k, F32), positive(7, m, n, F32)
    check(ops.dense(x, w), sums(x.t(), w.t()))
    dx, dw, _ = ops.dense_backward(dy, x, w, need_db=False)
    check(dx, sums(dy.t(), w))
    check(dw, sums(dy, x))
    ops.poll()
