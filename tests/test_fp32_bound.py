"""What the bound on fp32 products of one sign (tests/test_gpu_long_sums.py) lets
through, by emulation on the CPU: the kernel's scheme, and neither a product with
its low halves left out nor sums left in a truncating accumulator."""
import os
import sys

import numpy as np
import pytest

pytest.importorskip("torch")
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_long_sums import F32, LOSS, U  # noqa: E402
from test_gpu_ops import DENSE_MKN  # noqa: E402

BOUND = LOSS[F32] + 1.001 * U[F32]
K = sorted({d for mkn in DENSE_MKN for d in mkn})  # each length is contracted by one of the three products


def tf32(v):
    return (v.view(np.uint32) & np.uint32(0xFFFFE000)).view(np.float32)


def low(v):
    return tf32(((v - tf32(v)).view(np.uint32) + np.uint32(0x1000)).view(np.float32))


def cut(v):
    """Toward zero to 24 bits."""
    f = v.astype(np.float32)
    return np.where(f.astype(np.float64) > v, np.nextafter(f, np.float32(0)), f).astype(np.float64)


def product(a, b, low_halves, chunk):
    """Rows' products as the tensor core makes them: 8 of K an update, the sum cut at each; a set goes to
    a register's fp32 sum every `chunk` of K."""
    n, k = a.shape
    pad = -k % 8
    a, b = (np.pad(t, ((0, 0), (0, pad))) for t in (a, b))
    terms = [(tf32(a), tf32(b))]
    if low_halves:
        terms += [(tf32(a), low(b)), (low(a), tf32(b))]
    total = np.zeros(n, np.float32)
    for k0 in range(0, k + pad, chunk):
        sets = [np.zeros(n), np.zeros(n)]
        for i in range(k0, min(k + pad, k0 + chunk), 8):
            for j, (p, q) in enumerate(terms):
                s = min(j, 1)
                sets[s] = cut(sets[s] + (p[:, i:i + 8].astype(np.float64) * q[:, i:i + 8]).sum(1))
        total += (sets[0].astype(np.float32) + sets[1].astype(np.float32))
    return total


def errors(k, low_halves, chunk, rows=200):
    rng = np.random.default_rng(k)
    a, b = ((rng.random((rows, k)) / 8).astype(np.float32) for _ in range(2))
    want = (a.astype(np.float64) * b).sum(1)
    return np.abs(product(a, b, low_halves, chunk) / want - 1).max()


@pytest.mark.parametrize("k", K)
def test_the_scheme_passes_and_plain_tf32_fails(k):
    k = min(k, 8192)  # longer sums only repeat
    assert errors(k, True, 256) <= BOUND
    assert errors(k, False, 256) > BOUND


@pytest.mark.parametrize("k", [4000, 8192])
def test_one_set_for_a_long_sum_fails(k):
    assert errors(k, True, 1 << 30) > BOUND
