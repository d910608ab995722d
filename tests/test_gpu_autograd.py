"""Autograd through the operators' torch binding: a result knows of the inputs that
require a gradient, and theirs are those of the backward calls."""
import importlib
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "gelu", "lrelu", "sigmoid"]


@pytest.fixture(scope="module")
def ops():
    return importlib.import_module("maxim-rs_b200.ops")


def rand(seed, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stats", [False, True])
def test_layer_norm(ops, dtype, stats):
    x = rand(1, 5, 7, 96, dtype=dtype).requires_grad_()
    scale, bias = rand(2, 96, scale=0.1, shift=1.0).requires_grad_(), rand(3, 1, 96).requires_grad_()
    out = ops.layer_norm(x, scale, bias, stats=stats)
    y = out[0] if stats else out
    dy = rand(4, 5, 7, 96, dtype=dtype)
    y.backward(dy)
    with torch.no_grad():
        want, mean, rstd = ops.layer_norm(x, scale, bias, stats=True)
        dx, dscale, dbias = ops.layer_norm_backward(dy, x, scale, mean, rstd)
    assert torch.equal(y, want) and not want.requires_grad
    assert torch.equal(x.grad, dx) and torch.equal(scale.grad, dscale) and torch.equal(bias.grad, dbias.view(1, 96))
    if stats:
        assert torch.equal(out[1], mean) and torch.equal(out[2], rstd)
        assert not out[1].requires_grad and not out[2].requires_grad


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [1, 40])
def test_dense(ops, dtype, act, m):
    x, w = rand(1, m, 48, dtype=dtype).requires_grad_(), rand(2, 80, 48, dtype=dtype, scale=0.2).requires_grad_()
    b, r = rand(3, 80, dtype=dtype).requires_grad_(), rand(4, m, 80, dtype=dtype).requires_grad_()
    y = ops.dense(x, w, b, act=act, residual=r)
    dy = rand(5, m, 80, dtype=dtype)
    y.backward(dy)
    with torch.no_grad():
        want, pre = ops.dense(x, w, b, act=act, residual=r, save_pre=True)
        grads = ops.dense_backward(dy, x, w, pre=pre, act=act)
    assert torch.equal(y, want)
    assert all(torch.equal(t.grad, g) for t, g in zip((x, w, b, r), grads + (dy,)))
    y2, pre2 = ops.dense(x, w, b, act=act, residual=r, save_pre=True)
    assert y2.requires_grad and not pre2.requires_grad and torch.equal(pre2, pre)


def test_only_what_is_asked_for(ops):
    x, w, b = rand(1, 40, 48), rand(2, 80, 48), rand(3, 80)
    dy = rand(4, 40, 80)
    assert not ops.dense(x, w, b).requires_grad
    for i in range(3):
        t = [x.clone(), w.clone(), b.clone()]
        t[i].requires_grad_()
        ops.dense(*t, act="gelu").backward(dy)
        assert [v.grad is not None for v in t] == [j == i for j in range(3)]
    r = rand(5, 40, 80).requires_grad_()
    ops.dense(x, w, residual=r).backward(dy)
    assert torch.equal(r.grad, dy)
    for i in range(3):
        t = [rand(6, 9, 32), rand(7, 32), rand(8, 32)]
        t[i].requires_grad_()
        ops.layer_norm(*t).sum().backward()  # an expanded gradient
        assert [v.grad is not None for v in t] == [j == i for j in range(3)]
    with torch.no_grad():
        assert not ops.dense(x.requires_grad_(), w).requires_grad


def test_a_block_against_torch(ops):
    """Norm, two products and a residual, in fp32, against torch's own gradients in 64 bits: sums of
    a few hundred terms, 1e-5 of each gradient's size."""
    p = {"x": rand(1, 150, 40), "scale": rand(2, 40, scale=0.1, shift=1.0), "shift": rand(3, 40), "b1": rand(5, 160),
         "w1": rand(4, 160, 40, scale=0.15), "w2": rand(6, 40, 160, scale=0.08), "b2": rand(7, 40)}
    v = rand(8, 150, 40)
    mine = {k: t.clone().requires_grad_() for k, t in p.items()}
    n = ops.layer_norm(mine["x"], mine["scale"], mine["shift"])
    h = ops.dense(n, mine["w1"], mine["b1"], act="gelu")
    (ops.dense(h, mine["w2"], mine["b2"], residual=mine["x"]) * v).sum().backward()
    other = {k: t.double().requires_grad_() for k, t in p.items()}
    n = torch.nn.functional.layer_norm(other["x"], (40,), other["scale"], other["shift"], 1e-6)
    h = torch.nn.functional.gelu(n @ other["w1"].t() + other["b1"])
    ((other["x"] + h @ other["w2"].t() + other["b2"]) * v).sum().backward()
    for k in p:
        assert (mine[k].grad.double() - other[k].grad).norm() <= 1e-5 * other[k].grad.norm(), k


def test_second_gradients_are_refused(ops):
    x, w = rand(1, 40, 48).requires_grad_(), rand(2, 80, 48).requires_grad_()
    (dx,) = torch.autograd.grad(ops.dense(x, w, act="gelu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_a_wait_given_up_is_told_by_the_backward_pass(ops, mx):
    """Autograd runs it on a thread of its own, on which nobody can poll: the error is raised once."""
    x, w = rand(1, 40, 48).requires_grad_(), rand(2, 80, 48).requires_grad_()
    ops.dense(x, w).sum().backward()  # that thread has made a call
    y = ops.dense(x, w).sum()
    assert mx.lib().mx_dense_wait_check(2000, torch.cuda.current_stream().cuda_stream) == mx._native.MX_OK
    torch.cuda.synchronize()
    with pytest.raises(mx.MaximError, match="gave up a wait"):
        y.backward()
    with pytest.raises(mx.MaximError, match="gave up a wait"):
        ops.dense(x, w)
    with pytest.raises(mx.MaximError, match="gave up a wait"):
        ops.poll()
    x.grad = None
    ops.dense(x, w).sum().backward()
    assert torch.allclose(x.grad, w.detach().sum(0).expand(40, 48), rtol=1e-5, atol=1e-4)
    ops.poll()


def test_threads_train_on_one_stream(ops):
    """Forward calls on this thread while autograd's own thread runs another's backward pass."""
    x, w = rand(1, 700, 512, dtype=torch.bfloat16), rand(2, 1000, 512, dtype=torch.bfloat16, scale=0.03)
    dy = rand(3, 700, 1000, dtype=torch.bfloat16)

    def grads():
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        ops.dense(a, b, act="gelu").backward(dy)
        return a.grad, b.grad

    want, errors = grads(), []

    def work():
        try:
            for _ in range(30):
                if not all(torch.equal(a, b) for a, b in zip(grads(), want)):
                    raise AssertionError("gradients differ")
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
