"""The operators on the caller's device tensors (`maxim-rs_b200/ops.py`): layer
norm and the dense product, forward and backward, against plain 64-bit forms
of their formulas at the sizes and layouts where they can go wrong.

Tolerances are elementwise bounds from the arithmetic. U[t] is a type's unit
roundoff: a result is rounded once to its type, U[t] |y|. Sums run in fp32:
a sum of terms s with at most d roundings in any term's path is off by
d 2^-23 sum |s| (2^-23, not 2^-24: the tensor cores' accumulators truncate).
"""
import ctypes
import importlib
import math
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}  # where a type's steps stop shrinking
E32 = 2.0 ** -23
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = [F32, BF16, F16]
SLOPE = 0.2


@pytest.fixture(scope="module")
def ops():
    return importlib.import_module("maxim-rs_b200.ops")


def rand(seed, *shape, dtype=F32, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)


def close(got, want, tol, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got.double()).all(), what
    over = (got.double() - want).abs() - (tol + U[got.dtype] * want.abs() * 1.001 + TINY[got.dtype])
    assert got.numel() == 0 or over.max().item() <= 0, (what, over.max().item())


# ------------------------------------------------------------- layer norm
# Elements of a row that one thread adds before the tree: at most 32, the long
# rows' loops c / 512.
def ln_depth(c):
    return max(32, c / 512) + 24


def ln_exact(x, scale, bias, eps):
    x, scale, bias = x.double(), scale.double(), bias.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    return (x - mean) * rstd * scale + bias, mean, rstd


def check_ln(ops, x, scale, bias, eps=1e-6):
    y, mean, rstd = ops.layer_norm(x, scale, bias, eps=eps, stats=True)
    assert torch.equal(y, ops.layer_norm(x, scale, bias, eps=eps))
    wy, wm, wr = ln_exact(x, scale, bias, eps)
    c = x.shape[-1]
    d = ln_depth(c) * E32
    em = d * x.double().abs().mean(-1, keepdim=True)  # of the mean
    dev = (x.double() - wm).abs()
    # of rstd, relative: the sum of squares', and the mean's error in each deviation
    er = d + em * wr * (dev.mean(-1, keepdim=True) * wr + em * wr) + 4 * E32
    close(mean, wm.squeeze(-1), em.squeeze(-1), "mean")
    close(rstd, wr.squeeze(-1), (wr * er).squeeze(-1), "rstd")
    n = dev * wr
    close(y, wy, scale.double().abs() * (em * wr + n * (er + 4 * E32)) + 2 * E32 * bias.double().abs(), "y")


LN_C = [1, 2, 3, 4, 8, 24, 31, 32, 64, 100, 257, 512, 520, 769, 1024, 2048, 2056, 4096, 6000, 8192, 8200, 16384, 20000,
        20001]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", LN_C)
def test_layer_norm(ops, c, dtype):
    for i, rows in enumerate((1, 2, 7, 33, 600)):
        pt = dtype if i % 2 else F32
        x = rand(c + rows, rows, c, dtype=dtype, scale=1.5, shift=0.3)
        check_ln(ops, x, rand(1, c, dtype=pt, scale=0.1, shift=1.0), rand(2, c, dtype=pt, scale=0.1))


def ln_backward_exact(dy, x, scale, mean, rstd):
    dy, x, scale, mean, rstd = (t.double() for t in (dy, x, scale, mean.unsqueeze(-1), rstd.unsqueeze(-1)))
    n = (x - mean) * rstd
    g = dy * scale
    mg, mgn = g.mean(-1, keepdim=True), (g * n).mean(-1, keepdim=True)
    c = x.shape[-1]
    tol = rstd * E32 * (ln_depth(c) + 16) * (g.abs() + g.abs().mean(-1, keepdim=True) +
                                             n.abs() * (g * n).abs().mean(-1, keepdim=True))
    return rstd * (g - mg - n * mgn), (dy * n).reshape(-1, c), dy.reshape(-1, c), tol


def check_ln_backward(ops, dy, x, scale, mean, rstd):
    dx, ds, db = ops.layer_norm_backward(dy, x, scale, mean, rstd)
    wdx, ts, tb, tol = ln_backward_exact(dy, x, scale, mean, rstd)
    close(dx, wdx, tol, "dx")
    # Rows are added in a block, over blocks, and in two trees.
    depth = (ts.shape[0] / 148 + 200) * E32
    close(ds, ts.sum(0), depth * ts.abs().sum(0), "dscale")
    close(db, tb.sum(0), depth * tb.abs().sum(0), "dbias")
    again = ops.layer_norm_backward(dy, x, scale, mean, rstd)
    assert all(torch.equal(a, b) for a, b in zip((dx, ds, db), again))
    only, none, none2 = ops.layer_norm_backward(dy, x, scale, mean, rstd, need_params=False)
    assert torch.equal(only, dx) and none is None and none2 is None
    none, ds2, db2 = ops.layer_norm_backward(dy, x, scale, mean, rstd, need_dx=False)
    assert none is None and torch.equal(ds2, ds) and torch.equal(db2, db)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", LN_C)
def test_layer_norm_backward(ops, c, dtype):
    for i, rows in enumerate((1, 2, 9, 67, 3000)):
        pt = dtype if i % 2 else F32
        x = rand(c + rows, rows, c, dtype=dtype, scale=1.5, shift=0.3)
        _, mean, rstd = ln_exact(x, torch.ones(c, device="cuda"), torch.zeros(c, device="cuda"), 1e-6)
        check_ln_backward(ops, rand(7, rows, c, dtype=dtype), x, rand(1, c, dtype=pt, scale=0.1, shift=1.0),
                          mean.float().squeeze(-1), rstd.float().squeeze(-1))


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_layouts(ops, dtype):
    """Channel ranges of wider tensors (aligned and not), leading dimensions,
    transposes, expanded gradients."""
    c = 96
    scale, bias = rand(1, c, shift=1.0, scale=0.1), rand(2, c)
    wide = rand(3, 5, 7, 4 * c, dtype=dtype)
    for x in (wide[..., c:2 * c], wide[..., 3:3 + c], wide[:, ::2, :c], wide[..., ::4], wide[:, 0, 5:5 + c],
              rand(4, c, 50, dtype=dtype).t(), rand(5, 1, 3, c, dtype=dtype)[:, :, :], rand(6, c, dtype=dtype)):
        check_ln(ops, x, scale, bias)
        _, mean, rstd = ops.layer_norm(x, scale, bias, stats=True)
        assert mean.shape == x.shape[:-1]
        check_ln_backward(ops, rand(8, *x.shape, dtype=dtype), x, scale, mean, rstd)
        check_ln_backward(ops, torch.ones((), dtype=dtype, device="cuda").expand(x.shape), x, scale, mean, rstd)


def test_layer_norm_hard_values(ops):
    """Rows of one value, rows far from zero, an infinite value, a NaN: each row keeps to itself."""
    c = 512
    one, zero = torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")
    x = rand(1, 6, c)
    x[1] = 3.25
    x[2] += 1e4
    clean = ops.layer_norm(x, one, zero)
    assert torch.equal(clean[1], zero)
    check_ln(ops, x, one, zero)
    x[3, 17] = float("inf")
    x[4, 5] = float("nan")
    y, mean, rstd = ops.layer_norm(x, one, zero, stats=True)
    assert torch.isnan(y[3:5]).any(1).all()
    assert torch.equal(y[[0, 1, 2, 5]], clean[[0, 1, 2, 5]])
    assert torch.isnan(mean[4]) and torch.isinf(mean[3])


def test_layer_norm_no_rows(ops):
    x = torch.empty(0, 64, device="cuda")
    p = torch.ones(64, device="cuda")
    y, mean, rstd = ops.layer_norm(x, p, p, stats=True)
    assert y.shape == (0, 64) and mean.shape == (0,)
    dx, ds, db = ops.layer_norm_backward(x, x, p, mean, rstd)
    assert dx.shape == (0, 64) and not ds.any() and not db.any()


# ------------------------------------------------------------------ dense
def act64(v, act):
    if act == "gelu":
        return v * 0.5 * torch.erfc(-v / math.sqrt(2.0))
    if act == "lrelu":
        return torch.where(v >= 0, v, SLOPE * v)
    if act == "sigmoid":
        return torch.sigmoid(v)
    return v


def act_grad64(v, act):
    if act == "gelu":
        return 0.5 * torch.erfc(-v / math.sqrt(2.0)) + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    if act == "lrelu":
        return torch.where(v >= 0, 1.0, SLOPE).double()
    if act == "sigmoid":
        return torch.sigmoid(v) * torch.sigmoid(-v)
    return torch.ones_like(v)


def mm_error(dtype, k):
    """Of a sum of k products against the sum of their sizes. 16-bit products are
    exact; an accumulator is rounded once per 16 (fp32: 8, two regions). The
    fp32 split drops lo lo and rounds both lo: 3 * 2^-21 of a product."""
    if dtype is F32:
        return (k / 4 + 32) * E32 + 3 * 2.0 ** -21
    return (k / 16 + 32) * E32


def check_dense(ops, x, w, bias, act="none", residual=None):
    y, pre = ops.dense(x, w, bias, act=act, slope=SLOPE, residual=residual, save_pre=True)
    assert torch.equal(y, ops.dense(x, w, bias, act=act, slope=SLOPE, residual=residual))
    k = x.shape[-1]
    xd, wd = x.double(), w.double()
    wpre = xd @ wd.t()
    size = xd.abs() @ wd.abs().t()
    if bias is not None:
        wpre, size = wpre + bias.double(), size + bias.double().abs()
    e = mm_error(x.dtype, k) * size
    close(pre, wpre, e, "pre")
    want = act64(wpre, act)
    if residual is not None:
        want = want + residual.double()
        e = e + E32 * residual.double().abs()
    # No activation here is steeper than 1.13; their own evaluation is within
    # 4 ulp of max(1, |pre|).
    close(y, want, 1.13 * e + 4 * E32 * (1 + wpre.abs()), "y")


ACTS = ["none", "gelu", "lrelu", "sigmoid"]
# Few rows (the FMA kernel), one tile and less, ragged tiles, split sums, odd and unaligned sizes, depth.
DENSE_MKN = [(1, 1, 1), (1, 4096, 1000), (2, 31, 7), (3, 520, 8000), (4, 64, 64), (5, 513, 130), (8, 1024, 333),
             (9, 64, 64), (16, 5, 3), (33, 96, 40), (128, 64, 64), (129, 65, 257), (200, 1000, 1000), (64, 8192, 128),
             (517, 1023, 771), (1000, 128, 256), (2500, 72, 31), (300, 3000, 2049), (70000, 16, 24), (4000, 512, 1536),
             (100, 300, 40000), (2048, 1032, 1100)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mkn", DENSE_MKN)
def test_dense(ops, mkn, dtype):
    m, k, n = mkn
    act = ACTS[(m + k + n) % 4]
    x, w = rand(m, m, k, dtype=dtype), rand(n + 1, n, k, dtype=dtype, scale=1 / math.sqrt(k))
    check_dense(ops, x, w, rand(3, n, dtype=dtype), act, rand(4, m, n, dtype=dtype))
    check_dense(ops, x, w, None, ACTS[(m + k + n + 1) % 4])
    ops.poll()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_dense_activations(ops, act, dtype):
    for m in (3, 40):
        check_dense(ops, rand(1, m, 48, dtype=dtype, scale=2.0), rand(2, 80, 48, dtype=dtype, scale=0.5),
                    rand(3, 80, dtype=dtype), act)


@pytest.mark.parametrize("dtype", DTYPES)
def test_dense_layouts(ops, dtype):
    wide = rand(1, 4, 9, 256, dtype=dtype)
    w = rand(2, 48, 256, dtype=dtype, scale=0.1)
    bias = rand(3, 96, dtype=dtype)[::2]
    for x, ww in ((wide[..., 64:128], w[:, :64]), (wide[..., 3:67], w[:, 5:69]), (wide[..., ::4], w[:, ::4]),
                  (wide[:, 0, :100], w[:, 100:200]), (wide[0, 0], w), (rand(5, 256, 50, dtype=dtype).t(), w),
                  (wide[1:2, 3:4, :64], w[:, :64])):
        residual = rand(4, *x.shape[:-1], 100, dtype=dtype)[..., 7:55]
        check_dense(ops, x, ww, bias, "gelu", residual)
        check_dense_backward(ops, rand(6, *x.shape[:-1], 60, dtype=dtype)[..., 1:49], x, ww, "none", None)
        pre = rand(8, *x.shape[:-1], 64, dtype=dtype)[..., 8:56]
        check_dense_backward(ops, rand(7, *x.shape[:-1], 48, dtype=dtype), x, ww, "sigmoid", pre)
        ones = torch.ones((), dtype=dtype, device="cuda").expand(x.shape[:-1] + (48,))
        check_dense_backward(ops, ones, x, ww, "gelu", pre)


def check_dense_backward(ops, dy, x, w, act, pre):
    dx, dw, db = ops.dense_backward(dy, x, w, pre=pre, act=act, slope=SLOPE)
    n, k = w.shape
    dyd, xd, wd = dy.double().reshape(-1, n), x.double().reshape(-1, k), w.double()
    m = dyd.shape[0]
    d = dyd * act_grad64(pre.double().reshape(-1, n), act) if act != "none" else dyd
    # d's own error: the activation's derivative (6 ulp of 1 + |pre| covers the
    # four) and, with an activation, the rounding to the operands' type.
    e32 = 0 * d if act == "none" else dyd.abs() * (6 * E32 * (1 + pre.double().reshape(-1, n).abs()))
    e = e32 if act == "none" else e32 + U[dy.dtype] * d.abs() + TINY[dy.dtype]
    close(dx.reshape(-1, k), d @ wd, (e + mm_error(dy.dtype, n) * d.abs()) @ wd.abs(), "dx")
    close(dw, d.t() @ xd, (e + mm_error(dy.dtype, m) * d.abs()).t() @ xd.abs(), "dw")
    close(db, d.sum(0), (e32 + (m / 148 + 200) * E32 * d.abs()).sum(0), "db")
    again = ops.dense_backward(dy, x, w, pre=pre, act=act, slope=SLOPE)
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), again))
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0)):
        part = ops.dense_backward(dy, x, w, pre=pre, act=act, slope=SLOPE, need_dx=need[0], need_dw=need[1],
                                  need_db=need[2])
        for want, got, on in zip((dx, dw, db), part, need):
            assert torch.equal(got, want) if on else got is None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mkn", DENSE_MKN)
def test_dense_backward(ops, mkn, dtype):
    m, k, n = mkn
    x, w = rand(m, m, k, dtype=dtype), rand(n + 1, n, k, dtype=dtype, scale=1 / math.sqrt(k))
    dy = rand(5, m, n, dtype=dtype)
    act = ACTS[(m + k + n) % 4]
    for a in {act, "none"}:
        check_dense_backward(ops, dy, x, w, a, rand(6, m, n, dtype=dtype) if a != "none" else None)
    ops.poll()


@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(ops, act):
    """Central differences of a 64-bit loss sum(v * y) of norm, product, activation and residual, along a
    random direction of each input. The 64-bit difference is within 1e-7 of the derivative (h^2 of a
    third derivative, and rounding over h); the fp32 gradients within 1e-4 of the sum's size, from
    the bounds above over these lengths."""
    rows, c, n = 37, 48, 40
    x, scale, bias = rand(1, rows, c), rand(2, c, scale=0.1, shift=1.0), rand(3, c)
    w, b, res, v = rand(4, n, c, scale=0.15), rand(5, n), rand(6, rows, n), rand(7, rows, n)
    h, mean, rstd = ops.layer_norm(x, scale, bias, stats=True)
    y, pre = ops.dense(h, w, b, act=act, slope=SLOPE, residual=res, save_pre=True)
    dh, dw, db = ops.dense_backward(v, h, w, pre=pre, act=act, slope=SLOPE)
    dx, dscale, dbias = ops.layer_norm_backward(dh, x, scale, mean, rstd)

    def loss(x, scale, bias, w, b, res):
        hh = ln_exact(x, scale, bias, 1e-6)[0]
        return (v.double() * (act64(hh @ w.t() + b, act) + res)).sum()

    args = [t.double() for t in (x, scale, bias, w, b, res)]
    for i, grad in enumerate((dx, dscale, dbias, dw, db, v)):
        step = rand(20 + i, *args[i].shape).double()
        eps = 1e-6
        if act == "lrelu":
            eps = 1e-9  # short enough that no pre-activation crosses the kink
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + eps * step, args[i] - eps * step
        want = (loss(*up) - loss(*down)) / (2 * eps)
        got = (grad.double() * step).sum()
        size = (grad.double() * step).abs().sum()
        assert abs(got - want) <= 1e-4 * size, (act, i, got.item(), want.item())


def test_dense_hard_values(ops):
    """Infinite and NaN inputs stay in their own rows and columns; large 16-bit
    sums overflow to infinity, not to something else."""
    for dtype in DTYPES:
        for m in (6, 140):
            x, w = rand(1, m, 96, dtype=dtype), rand(2, 72, 96, dtype=dtype)
            clean = ops.dense(x, w)
            x2, w2 = x.clone(), w.clone()
            x2[1, 5] = float("inf")
            x2[2, 7] = float("nan")
            w2[3, 1] = float("nan")
            y = ops.dense(x2, w2)
            assert not torch.isfinite(y[1]).any() and torch.isnan(y[2]).all() and torch.isnan(y[:, 3]).all()
            rows, cols = [i for i in range(m) if i not in (1, 2)], [j for j in range(72) if j != 3]
            assert torch.equal(y[rows][:, cols], clean[rows][:, cols])
    big = torch.full((20, 64), 60000.0, dtype=F16, device="cuda")
    assert torch.isinf(ops.dense(big, torch.ones(8, 64, dtype=F16, device="cuda"))).all()


@pytest.mark.parametrize("m", [9, 40, 300])
@pytest.mark.parametrize("other", [1.0, 1.1, -0.3, 2.0 ** -20])  # exact in TF32, and with low bits
def test_infinite_operands_in_fp32(ops, m, other):
    """From the tensor cores an infinite fp32 operand gives NaN wherever it is used, whatever it
    meets; one or two rows give what IEEE does."""
    for inf in (float("inf"), -float("inf")):
        x, w = torch.full((m, 64), other, device="cuda"), torch.full((48, 64), other, device="cuda")
        x[1, 5] = inf
        w[7, 9] = inf
        hit = torch.zeros(m, 48, dtype=torch.bool, device="cuda")
        hit[1], hit[:, 7] = True, True
        assert torch.equal(torch.isnan(ops.dense(x, w)), hit)
        few = ops.dense(x[:2], w)
        assert torch.isinf(few[1]).all() and torch.isinf(few[:, 7]).all()
        dy = torch.full((m, 48), other, device="cuda")
        dy[3, 2] = inf
        dx, dw, db = ops.dense_backward(dy, x, w)
        assert torch.isnan(dx[3]).all() and torch.isnan(dx[:, 9]).all()
        assert torch.isfinite(dx[[0, 2, 4]][:, :9]).all()
        assert torch.isnan(dw[2]).all() and torch.isnan(dw[:, 5]).all() and torch.isfinite(dw[3:, 6:]).all()
        assert torch.isinf(db[2]) and torch.isfinite(db[[0, 1, 3]]).all()


def test_activation_ends(ops):
    """Pre-activations of +-inf and +-1e30 through the activations and their gradients."""
    inf = float("inf")
    v = torch.tensor([[inf], [-inf], [1e30], [-1e30], [0.0], [-0.0]], device="cuda")
    one = torch.ones(1, 1, device="cuda")
    dy = torch.ones_like(v)
    for act, y, g in (("gelu", [inf, 0, 1e30, 0, 0, 0], [1, 0, 1, 0, 0.5, 0.5]),
                      ("lrelu", [inf, -inf, 1e30, -2e29, 0, 0], [1, 0.2, 1, 0.2, 1, 1]),
                      ("sigmoid", [1, 0, 1, 0, 0.5, 0.5], [0, 0, 0, 0, 0.25, 0.25])):
        want = torch.tensor(y, device="cuda", dtype=F32)
        assert torch.allclose(ops.dense(v, one, act=act, slope=SLOPE).flatten(), want, rtol=1e-6, atol=0), act
        _, _, db = ops.dense_backward(dy, torch.zeros_like(v), one, pre=v, act=act, slope=SLOPE)
        assert abs(db.item() - sum(g)) < 1e-5, act
        for i in range(6):
            _, _, db = ops.dense_backward(dy[i:i + 1], one, one, pre=v[i:i + 1], act=act, slope=SLOPE)
            assert abs(db.item() - g[i]) < 1e-6, (act, i)


def test_dense_no_rows(ops):
    x, w = torch.empty(0, 64, device="cuda"), torch.ones(32, 64, device="cuda")
    assert ops.dense(x, w).shape == (0, 32)
    dx, dw, db = ops.dense_backward(torch.empty(0, 32, device="cuda"), x, w)
    assert dx.shape == (0, 64) and dw.shape == (32, 64) and not dw.any() and not db.any()


def test_other_streams(ops):
    """Calls on a side stream are ordered by that stream alone."""
    x, w = rand(1, 4000, 1023, dtype=BF16), rand(2, 900, 1023, dtype=BF16, scale=0.03)
    want = ops.dense(x, w, act="gelu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    outs = []
    with torch.cuda.stream(s):
        for _ in range(4):
            outs.append(ops.dense(x, w, act="gelu"))
    s.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def overlapping_calls(ops):
    """Calls that hand data on through their workspace: unaligned copies, split sums, the activation's gradient."""
    def forward(seed, m, k, n):
        x, w = rand(seed, m, k, dtype=BF16), rand(seed + 1, n, k, dtype=BF16, scale=0.03)
        return lambda: (ops.dense(x, w, act="gelu"),)

    def backward(seed, m, k, n):
        x, w = rand(seed, m, k, dtype=BF16), rand(seed + 1, n, k, dtype=BF16, scale=0.03)
        dy, pre = rand(seed + 2, m, n, dtype=BF16), rand(seed + 3, m, n, dtype=BF16)
        return lambda: ops.dense_backward(dy, x, w, pre=pre, act="gelu")

    def norm(seed, rows, c):
        x, dy = rand(seed, rows, c), rand(seed + 1, rows, c)
        _, mean, rstd = ops.layer_norm(x, dy[0], dy[1], stats=True)
        return lambda: ops.layer_norm_backward(dy, x, dy[0], mean, rstd)

    return [forward(1, 300, 1023, 900), backward(11, 700, 512, 1000), norm(21, 3000, 257), forward(31, 64, 8192, 128),
            backward(41, 90, 333, 77), backward(51, 2500, 256, 264)]


def test_threads_on_one_stream(ops):
    """Host threads that call on the same stream at once get what serial calls give."""
    calls = overlapping_calls(ops)
    want = [[t.clone() for t in c()] for c in calls]
    torch.cuda.synchronize()
    got, errors = [[] for _ in calls], []
    start = threading.Barrier(len(calls))

    def work(i):
        try:
            start.wait()
            for _ in range(40):
                got[i].append(calls[i]())
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for i, results in enumerate(got):
        assert len(results) == 40
        for r in results:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i])), i


def test_streams_in_flight_together(ops):
    """Calls issued in turn on several streams, all of them at work at the same time."""
    calls = overlapping_calls(ops)
    want = [[t.clone() for t in c()] for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(calls[i]())
    torch.cuda.synchronize()
    for i, results in enumerate(got):
        for r in results:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i])), i


def test_a_wait_given_up(ops, mx):
    """A wait that runs out leaves a record: dense calls are refused on every thread
    until that thread has polled, the norm is not, and afterwards all is as before."""
    x, w = rand(1, 40, 64), rand(2, 48, 64)
    want = ops.dense(x, w)
    ops.poll()
    lib, stream = mx.lib(), torch.cuda.current_stream().cuda_stream
    assert lib.mx_dense_wait_check(1000001, stream) == mx._native.MX_E_INVALID
    assert lib.mx_dense_wait_check(2000, stream) == mx._native.MX_OK
    torch.cuda.synchronize()
    for _ in range(2):
        with pytest.raises(mx.MaximError, match="gave up a wait"):
            ops.dense(x, w)
    with pytest.raises(mx.MaximError, match="gave up a wait"):
        ops.dense_backward(rand(3, 40, 48), x, w)
    ops.layer_norm(x, w[0], w[1])
    with pytest.raises(mx.MaximError, match="device 0 gave up a wait"):
        ops.poll()
    ops.poll()
    assert torch.equal(ops.dense(x, w), want)
    # Two threads: the one's poll leaves the record to the other.
    seen, used, left = [], threading.Event(), threading.Event()

    def other():
        ops.dense(x, w)
        used.set()
        left.wait(20)
        for call in (lambda: ops.dense(x, w), ops.poll, ops.poll, lambda: ops.dense(x, w)):
            try:
                call()
                seen.append("taken")
            except mx.MaximError:
                seen.append("refused")

    t = threading.Thread(target=other)
    t.start()
    assert used.wait(20)
    assert lib.mx_dense_wait_check(2000, stream) == mx._native.MX_OK
    torch.cuda.synchronize()
    with pytest.raises(mx.MaximError):
        ops.poll()
    left.set()
    t.join()
    assert seen == ["refused", "refused", "taken", "taken"]
    assert torch.equal(ops.dense(x, w), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_calls_read_what_the_call_before_wrote(ops, dtype):
    """Weights that the call just before made (its blocks may still be leaving) serve
    one token and several, over and over."""
    x, dy = rand(1, 64, 256, dtype=dtype), rand(2, 64, 512, dtype=dtype)
    token, few = rand(3, 1, 256, dtype=dtype), rand(4, 40, 256, dtype=dtype)
    signs = [1.0, -2.0, 0.5, -1.0]
    grads = [(dy * s).contiguous() for s in signs]
    want = []
    for g in grads:
        _, dw, _ = ops.dense_backward(g, x, x[:1].expand(512, 256).contiguous(), need_dx=False)
        torch.cuda.synchronize()
        want.append((ops.dense(token, dw), ops.dense(few, dw)))
        torch.cuda.synchronize()
    w = x[:1].expand(512, 256).contiguous()
    got = []
    for _ in range(50):
        for g in grads:
            _, dw, _ = ops.dense_backward(g, x, w, need_dx=False)  # the allocator gives the same place again
            got.append((ops.dense(token, dw), ops.dense(few, dw)))
            del dw
    for i, r in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(r, want[i % 4])), i


def test_graph_capture(ops):
    """The calls can be captured (they allocate through torch's graph pool only)."""
    x, w = rand(1, 300, 1023, dtype=BF16), rand(2, 900, 1023, dtype=BF16, scale=0.03)
    scale = torch.ones(1023, device="cuda")
    want = ops.dense(ops.layer_norm(x, scale, scale), w, act="gelu")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.dense(ops.layer_norm(x, scale, scale), w, act="gelu")
    got.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def c_call(mx, ops, entry, layout, values, ws_at=None):
    """A call through the C ABI, its workspace filled with NaN bytes."""
    ws = None
    if ws_at is not None:
        need = ctypes.c_int64()
        mx._native.check(getattr(mx.lib(), entry + "_workspace")(layout.pack(*values), ctypes.byref(need)))
        ws = torch.full((need.value + 16,), 255, dtype=torch.uint8, device="cuda")
        values[ws_at], values[ws_at + 1] = ws.data_ptr(), need.value
    mx._native.check(getattr(mx.lib(), entry)(layout.pack(*values), torch.cuda.current_stream().cuda_stream))
    return ws


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [5, 8])  # unaligned and aligned rows of the outputs
def test_strided_outputs_and_in_place_results(mx, ops, dtype, gap):
    """The C ABI's output strides: what lies between the rows stays, at every size; and results over their inputs."""
    code = ops._DT[dtype]
    for m, k, n in ((1, 64, 48), (40, 72, 48), (300, 200, 136), (700, 1000, 264), (64, 4096, 64)):
        x, w = rand(1, m, k, dtype=dtype), rand(2, n, k, dtype=dtype, scale=1 / math.sqrt(k))
        res, dy = rand(3, m, n, dtype=dtype), rand(4, m, n, dtype=dtype)
        want, want_pre = ops.dense(x, w, act="gelu", residual=res, save_pre=True)
        y, pre = (torch.full((m, n + gap), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        y[:, :n] = res  # the residual's place becomes the result's
        P = torch.Tensor.data_ptr
        keep = c_call(mx, ops, "mx_dense", ops._DENSE, [P(x), P(w), 0, P(y), P(y), P(pre), 0, 0, m, k, n, k, k, n + gap,
                                                        n + gap, n + gap, code, 1, 0.0, 0], 6)
        assert torch.equal(y[:, :n], want) and torch.equal(pre[:, :n], want_pre), (m, k, n)
        assert (y[:, n:] == 7).all() and (pre[:, n:] == 7).all()
        dx, dw = (torch.full((r, k + gap), 7.0, dtype=dtype, device="cuda") for r in (m, n))
        db = torch.empty(n, dtype=dtype, device="cuda")
        keep2 = c_call(mx, ops, "mx_dense_backward", ops._DENSE_BACKWARD,
                       [P(dy), P(x), P(w), P(want_pre), P(dx), P(dw), P(db), 0, 0, m, k, n, n, k, k, n, k + gap, k + gap,
                        code, 1, 0.0, 0], 7)
        got = ops.dense_backward(dy, x, w, pre=want_pre, act="gelu")
        assert all(torch.equal(a, b) for a, b in zip((dx[:, :k], dw[:, :k], db), got)), (m, k, n)
        assert (dx[:, k:] == 7).all() and (dw[:, k:] == 7).all()
        scale, bias = rand(5, k, shift=1.0), rand(6, k)
        want, mean, rstd = ops.layer_norm(x, scale, bias, stats=True)
        z = torch.full((m, k + gap), 7.0, dtype=dtype, device="cuda")
        z[:, :k] = x
        c_call(mx, ops, "mx_layer_norm", ops._NORM,
               [P(z), P(scale), P(bias), P(z), 0, 0, m, k, k + gap, k + gap, code, 0, 1e-6, 0])
        # Unaligned rows are summed in another order.
        close(z[:, :k], want.double(), 1e-5 * (1 + want.double().abs()) + 2 * U[dtype] * want.double().abs(), "in place")
        assert (z[:, k:] == 7).all()
        g = rand(7, m, k, dtype=dtype)
        want = ops.layer_norm_backward(g, x, scale, mean, rstd)[0]
        z[:, :k] = g
        c_call(mx, ops, "mx_layer_norm_backward", ops._NORM_BACKWARD,
               [P(z), P(x), P(scale), P(mean), P(rstd), P(z), 0, 0, 0, 0, m, k, k + gap, k, k + gap, code, 0], 8)
        close(z[:, :k], want.double(), 1e-5 * (1 + want.double().abs()) + 2 * U[dtype] * want.double().abs(), "in place")
        assert (z[:, k:] == 7).all()
        torch.cuda.synchronize()
        del keep, keep2


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_offsets_past_32_bits(ops, dtype):
    """A channel range of a tensor of 4.6e9 elements: the last rows lie past 2^32 of them."""
    wide = torch.empty(70000, 65536, dtype=dtype, device="cuda")
    x = wide[:, 60000:60096]
    x.copy_(rand(1, 70000, 96, dtype=dtype))
    scale, bias = rand(2, 96, scale=0.1, shift=1.0), rand(3, 96)
    check_ln(ops, x, scale, bias)
    _, mean, rstd = ops.layer_norm(x, scale, bias, stats=True)
    check_ln_backward(ops, x, x, scale, mean, rstd)
    w = rand(4, 40, 96, dtype=dtype, scale=0.1)
    check_dense(ops, x, w, None, "gelu", rand(5, 70000, 40, dtype=dtype))
    dy = wide[:, 50000:50040]
    dy.copy_(rand(6, 70000, 40, dtype=dtype))
    check_dense_backward(ops, dy, x, w, "none", None)


def test_refusals(ops, mx):
    x, w = torch.ones(4, 8, device="cuda"), torch.ones(6, 8, device="cuda")
    p = torch.ones(8, device="cuda")
    bad = [
        (ValueError, lambda: ops.layer_norm(x.cpu(), p, p)),
        (TypeError, lambda: ops.layer_norm(x.double(), p, p)),
        (TypeError, lambda: ops.layer_norm(x, p.half(), p.half())),
        (ValueError, lambda: ops.layer_norm(x, p[:7], p)),
        (mx.MaximError, lambda: ops.layer_norm(x, p, p, eps=-1.0)),
        (mx.MaximError, lambda: ops.layer_norm(x[:, :0], p[:0], p[:0])),
        (ValueError, lambda: ops.layer_norm_backward(x[:2], x, p, x[:, 0], x[:, 0])),
        (ValueError, lambda: ops.layer_norm_backward(x, x, p, x[:2, 0], x[:, 0])),
        (ValueError, lambda: ops.dense(x, w[:, :7])),
        (ValueError, lambda: ops.dense(x, w, p)),
        (ValueError, lambda: ops.dense(x, w, act="relu6")),
        (ValueError, lambda: ops.dense(x, w, residual=x)),
        (TypeError, lambda: ops.dense(x, w.half())),
        (ValueError, lambda: ops.dense(x, w.cpu())),
        (mx.MaximError, lambda: ops.dense(x[:, :0], w[:, :0])),
        (ValueError, lambda: ops.dense_backward(x, x, w)),
        (ValueError, lambda: ops.dense_backward(torch.ones(4, 6, device="cuda"), x, w, act="gelu")),
        (ValueError, lambda: ops.dense_backward(torch.ones(3, 6, device="cuda"), x, w)),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            pytest.fail("case %d was taken" % i)
