"""Operators on the caller's own CUDA tensors (torch): layer norm and the dense
product, each with its backward pass, over the C ABI (`mx_layer_norm`,
`mx_dense` and their `_backward` forms in include/maxim_b200.h).

The reference has only the forward forms, as ops of a plan; these calls are
for training or serving layers outside one. This module checks shapes, marshals
arguments and allocates outputs and workspaces with torch; the work is done by
the library's kernels on the current stream of the tensors' device. Calls
return without waiting. Tensors are fp32, bf16 or fp16; leading dimensions are
rows, the last is the row. A tensor whose rows lie apart (a channel range of a
wider one) is taken as it is; one that is no matrix of contiguous rows (a
transpose, an expanded gradient) is copied first.
"""
import struct

import torch

from . import _native

_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTS = {"none": 0, "gelu": 1, "lrelu": 2, "sigmoid": 3}

# The argument structs of include/maxim_b200.h.
_NORM = struct.Struct("<6Q4q2ifi")
_NORM_BACKWARD = struct.Struct("<9Q6q2i")
_DENSE = struct.Struct("<7Q9q2ifi")
_DENSE_BACKWARD = struct.Struct("<8Q10q2ifi")


def _rows(t, what, cols=None):
    """The tensor as a matrix of rows: (data pointer, rows, columns, row stride, the tensor kept alive)."""
    c = t.shape[-1] if t.dim() else 0
    if t.dim() == 2:
        rows = t.shape[0]
    else:
        if t.dim() == 0:
            raise ValueError("%s: a scalar has no rows" % what)
        rows = t.numel() // c if c else 0
    if cols is not None and c != cols:
        raise ValueError("%s: rows of %d elements, expected %d" % (what, c, cols))
    if rows <= 1:
        if c > 1 and t.stride(-1) != 1:
            t = t.contiguous()
        return t.data_ptr(), rows, c, c, t
    if t.dim() == 2:
        s = t.stride(0)
        if (t.stride(1) == 1 or c == 1) and s >= c:
            return t.data_ptr(), rows, c, s, t
    elif not t.is_contiguous():
        # Leading dimensions that step evenly through memory are rows too.
        lead = [(n, st) for n, st in zip(t.shape[:-1], t.stride()[:-1]) if n != 1]
        even = all(a_st == b_n * b_st for (_, a_st), (b_n, b_st) in zip(lead, lead[1:]))
        if even and (t.stride(-1) == 1 or c == 1) and lead[-1][1] >= c:
            return t.data_ptr(), rows, c, lead[-1][1], t
    t = t.contiguous()
    return t.data_ptr(), rows, c, c, t


def _device(t, *others):
    if not t.is_cuda:
        raise ValueError("the operators take CUDA tensors, got one on %s" % t.device)
    for o in others:
        if o is not None and o.device != t.device:
            raise ValueError("tensors on %s and %s" % (t.device, o.device))
    return t.device.index


def _dtype(t, *others):
    code = _DT.get(t.dtype)
    if code is None:
        raise TypeError("the operators take float32, bfloat16 or float16, got %s" % t.dtype)
    for o in others:
        if o is not None and o.dtype != t.dtype:
            raise TypeError("tensors of %s and %s" % (t.dtype, o.dtype))
    return code


def _params(dtype, c, *params):
    """The type code of the norm's parameter vectors: the tensors' own type, or fp32."""
    pt = params[0].dtype
    if pt is not dtype and pt is not torch.float32:
        raise TypeError("parameters of %s with tensors of %s" % (pt, dtype))
    return _DT[pt], [_vector(p, pt, c) for p in params]


def _vector(p, dtype, n):
    if p.dtype is not dtype:
        raise TypeError("a vector of %s, expected %s" % (p.dtype, dtype))
    if p.numel() != n:
        raise ValueError("a vector of %d elements, expected %d" % (p.numel(), n))
    return p if p.is_contiguous() else p.contiguous()


def _launch(entry, query, layout, ws_at, values, device):
    """Call `entry` on the device's current stream with the packed argument
    struct, giving it the workspace that `query` asks for."""
    lib = _native.lib()
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _launch(entry, query, layout, ws_at, values, device)
    if query is not None:
        need = _native.ctypes.c_int64()
        rc = getattr(lib, query)(layout.pack(*values), _native.ctypes.byref(need))
        if rc != 0:
            _native.check(rc)
        if need.value:
            ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
            values[ws_at] = ws.data_ptr()
            values[ws_at + 1] = need.value
    rc = getattr(lib, entry)(layout.pack(*values), torch.cuda.current_stream().cuda_stream)
    if rc != 0:
        _native.check(rc)


def layer_norm(x, scale, bias, eps=1e-6, stats=False):
    """(x - mean) * rstd * scale + bias over the last dimension. With `stats`
    also the fp32 mean and rstd of every row, which the backward pass takes:
    (y, mean, rstd). scale and bias are of x's type or fp32."""
    device, code = _device(x, scale, bias), _dtype(x)
    xp, rows, c, xs, x_ = _rows(x, "x")
    pcode, (scale, bias) = _params(x.dtype, c, scale, bias)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = rstd = None
    if stats:
        mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _launch("mx_layer_norm", None, _NORM, 0,
            (xp, scale.data_ptr(), bias.data_ptr(), y.data_ptr(), mean.data_ptr() if stats else 0,
             rstd.data_ptr() if stats else 0, rows, c, xs, c, code, pcode, eps, 0), device)
    return (y, mean, rstd) if stats else y


def layer_norm_backward(dy, x, scale, mean, rstd, need_dx=True, need_params=True):
    """The gradients of layer_norm: (dx, dscale, dbias), None where not needed.
    mean and rstd are the forward pass's."""
    device, code = _device(x, dy, scale, mean, rstd), _dtype(x, dy)
    xp, rows, c, xs, x_ = _rows(x, "x")
    if dy.shape != x.shape:
        raise ValueError("dy has shape %s, x %s" % (tuple(dy.shape), tuple(x.shape)))
    dyp, _, _, dys, dy_ = _rows(dy, "dy")
    pcode, (scale,) = _params(x.dtype, c, scale)
    mean, rstd = _vector(mean, torch.float32, rows), _vector(rstd, torch.float32, rows)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_dx else None
    dscale = torch.empty_like(scale) if need_params else None
    dbias = torch.empty_like(scale) if need_params else None
    _launch("mx_layer_norm_backward", "mx_layer_norm_backward_workspace" if need_params else None, _NORM_BACKWARD, 8,
            [dyp, xp, scale.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dx.data_ptr() if need_dx else 0,
             dscale.data_ptr() if need_params else 0, dbias.data_ptr() if need_params else 0, 0, 0, rows, c, dys, xs, c,
             code, pcode], device)
    return dx, dscale, dbias


def dense(x, w, bias=None, act="none", slope=0.2, residual=None, save_pre=False):
    """act(x @ w.T + bias) + residual: x [..., k], w [n, k], bias [n], residual
    [..., n]. act is one of "none", "gelu" (the erf form), "lrelu" (leaky, with
    `slope`), "sigmoid". With `save_pre` also x @ w.T + bias, which the backward
    pass of an activation takes: (y, pre)."""
    device, code = _device(x, w, bias, residual), _dtype(x, w, bias, residual)
    xp, m, k, xs, x_ = _rows(x, "x")
    if w.dim() != 2:
        raise ValueError("w has %d dimensions, expected 2" % w.dim())
    wp, n, _, ws, w_ = _rows(w, "w", k)
    shape = x.shape[:-1] + (n,)
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    pre = torch.empty(shape, dtype=x.dtype, device=x.device) if save_pre else None
    rp = rs = 0
    if residual is not None:
        if residual.shape != shape:
            raise ValueError("residual has shape %s, the product %s" % (tuple(residual.shape), tuple(shape)))
        rp, _, _, rs, r_ = _rows(residual, "residual")
    if bias is not None:
        bias = _vector(bias, x.dtype, n)
    _launch("mx_dense", "mx_dense_workspace", _DENSE, 6,
            [xp, wp, 0 if bias is None else bias.data_ptr(), rp, y.data_ptr(), pre.data_ptr() if save_pre else 0, 0, 0,
             m, k, n, xs, ws, rs, n, n, code, _act(act), slope, 0], device)
    return (y, pre) if save_pre else y


def dense_backward(dy, x, w, pre=None, act="none", slope=0.2, need_dx=True, need_dw=True, need_db=True):
    """The gradients of dense: (dx, dw, db), None where not needed. pre is the
    forward pass's (with an activation); the residual's gradient is dy."""
    device, code = _device(dy, x, w, pre), _dtype(dy, x, w, pre)
    dyp, m, n, dys, dy_ = _rows(dy, "dy")
    xp, mx, k, xs, x_ = _rows(x, "x")
    if w.dim() != 2 or w.shape[0] != n:
        raise ValueError("w has shape %s, dy rows of %d" % (tuple(w.shape), n))
    wp, _, _, ws, w_ = _rows(w, "w", k)
    if dy.shape[:-1] != x.shape[:-1]:
        raise ValueError("dy has shape %s, x %s" % (tuple(dy.shape), tuple(x.shape)))
    pp = ps = 0
    if act != "none":
        if pre is None or pre.shape != dy.shape:
            raise ValueError("the gradient of %s needs pre, of dy's shape" % act)
        pp, _, _, ps, p_ = _rows(pre, "pre")
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_dx else None
    dw = torch.empty((n, k), dtype=x.dtype, device=x.device) if need_dw else None
    db = torch.empty(n, dtype=x.dtype, device=x.device) if need_db else None
    _launch("mx_dense_backward", "mx_dense_backward_workspace", _DENSE_BACKWARD, 7,
            [dyp, xp, wp, pp, dx.data_ptr() if need_dx else 0, dw.data_ptr() if need_dw else 0,
             db.data_ptr() if need_db else 0, 0, 0, m, k, n, dys, xs, ws, ps, k, k, code, _act(act), slope, 0], device)
    return dx, dw, db


def _act(name):
    code = ACTS.get(name)
    if code is None:
        raise ValueError("act %r is not one of %s" % (name, ", ".join(ACTS)))
    return code


def poll():
    """`mx_dense_poll`: raise if a dense kernel finished so far gave up a wait
    in its pipeline (its output is then not to be used). Does not wait."""
    _native.check(_native.lib().mx_dense_poll(), "dense")
