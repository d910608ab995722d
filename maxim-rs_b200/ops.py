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
transpose, an expanded gradient) is copied first. Host threads may call at
once. layer_norm and dense are known to autograd; the backward calls are there
for programs that chain them by hand.
"""
import ctypes
import struct
import threading

import torch

from . import _native

# What torch.cuda.current_device, current_stream and is_current_stream_capturing
# ask, without their wrappers (4 us of a 12 us call).
_cuda_device = torch._C._cuda_getDevice
_cuda_stream = torch._C._cuda_getCurrentRawStream
_cuda_capturing = torch._C._cuda_isCurrentStreamCapturing

_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTS = {"none": 0, "gelu": 1, "lrelu": 2, "sigmoid": 3}

# The argument structs of include/maxim_b200.h.
_NORM = struct.Struct("<6Q4q2ifi")
_NORM_BACKWARD = struct.Struct("<9Q6q2i")
_DENSE = struct.Struct("<7Q9q2ifi")
_DENSE_BACKWARD = struct.Struct("<8Q10q2ifi")


def _rows(t, what, cols=None):
    """The tensor as a matrix of rows: (data pointer, rows, columns, row stride, the tensor to keep alive)."""
    shape = t.shape
    if not shape:
        raise ValueError("%s: a scalar has no rows" % what)
    c = shape[-1]
    if cols is not None and c != cols:
        raise ValueError("%s: rows of %d elements, expected %d" % (what, c, cols))
    rows = shape[0] if len(shape) == 2 else (t.numel() // c if c else 0)
    if t.is_contiguous():
        return t.data_ptr(), rows, c, c, t
    if t.stride(-1) == 1 or c == 1:
        # Leading dimensions that step evenly through memory are rows too.
        lead = [(n, st) for n, st in zip(shape[:-1], t.stride()[:-1]) if n != 1]
        if not lead:
            return t.data_ptr(), rows, c, c, t
        step = lead[-1][1]
        if step >= c and all(a[1] == b[0] * b[1] for a, b in zip(lead, lead[1:])):
            return t.data_ptr(), rows, c, step, t
    t = t.contiguous()
    return t.data_ptr(), rows, c, c, t


def _where(t, *others):
    """The device index of tensors that must all be on one CUDA device."""
    device = t.get_device()
    if device < 0:
        raise ValueError("the operators take CUDA tensors, got one on %s" % t.device)
    for o in others:
        if o is not None and o.get_device() != device:
            raise ValueError("tensors on %s and %s" % (t.device, o.device))
    return device


def _dtype(t, *others):
    dt = t.dtype
    if dt not in _DT:
        raise TypeError("the operators take float32, bfloat16 or float16, got %s" % dt)
    for o in others:
        if o is not None and o.dtype is not dt:
            raise TypeError("tensors of %s and %s" % (dt, o.dtype))
    return _DT[dt]


def _vector(p, dtype, n):
    if p.dtype is not dtype:
        raise TypeError("a vector of %s, expected %s" % (p.dtype, dtype))
    if p.numel() != n:
        raise ValueError("a vector of %d elements, expected %d" % (p.numel(), n))
    return p if p.is_contiguous() else p.contiguous()


def _param_dtype(p, dtype):
    """The norm's parameter vectors are of the tensors' own type or fp32."""
    if p.dtype is not dtype and p.dtype is not torch.float32:
        raise TypeError("parameters of %s with tensors of %s" % (p.dtype, dtype))
    return p.dtype


def _like(x):
    """A dense tensor of x's shape and type, by the quickest call."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _act(name):
    if name not in ACTS:
        raise ValueError("act %r is not one of %s" % (name, ", ".join(ACTS)))
    return ACTS[name]


# Workspaces up to _WS_KEEP bytes stay with the host thread and stream that they
# were made for. Not with the stream alone: a call issues several kernels that
# hand data on through its workspace, and does so without the interpreter's
# lock, so the kernels of two threads' calls may lie in a stream in any order.
# Larger ones, and those of a captured graph (which must own its memory), come
# from torch's allocator at each call.
_WS_KEEP = 32 << 20


class _Kept(threading.local):
    def __init__(self):
        self.by_stream = {}  # (device, stream): (tensor, address, bytes)


_kept = _Kept()


def _launch(entry, layout, values, device, ws_at=None):
    """Call `entry` on the device's current stream with the packed argument
    struct. With `ws_at` (the index of the workspace pointer) it may need a workspace."""
    lib = _native.lib()
    if device != _cuda_device():
        with torch.cuda.device(device):
            return _launch(entry, layout, values, device, ws_at)
    stream = _cuda_stream(device)
    if ws_at is None:
        return _native.check(getattr(lib, entry)(layout.pack(*values), stream))
    capturing = _cuda_capturing()
    # Held until the kernels are issued: from then on the stream's order protects it.
    kept = None if capturing else _kept.by_stream.get((device, stream))
    if kept is not None:
        values[ws_at], values[ws_at + 1] = kept[1], kept[2]
    rc = getattr(lib, entry)(layout.pack(*values), stream)
    if rc == _native.MX_OK:
        return
    if rc != _native.MX_E_INVALID:
        _native.check(rc)
    # Refused, perhaps only for the workspace: the query refuses too if not.
    need = ctypes.c_int64()
    _native.check(getattr(lib, entry + "_workspace")(layout.pack(*values), ctypes.byref(need)))
    if need.value <= values[ws_at + 1]:
        _native.check(rc)
    keep = need.value <= _WS_KEEP and not capturing
    size = max(need.value, 1 << 20) if keep else need.value
    ws = torch.empty(size, dtype=torch.uint8, device=torch.device("cuda", device))
    if keep:
        _kept.by_stream[device, stream] = (ws, ws.data_ptr(), size)
    values[ws_at], values[ws_at + 1] = ws.data_ptr(), size
    _native.check(getattr(lib, entry)(layout.pack(*values), stream))


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, scale, bias, eps):
        y, mean, rstd = layer_norm(x, scale, bias, eps, stats=True)
        ctx.save_for_backward(x, scale, mean, rstd)
        ctx.bias_shape = bias.shape
        ctx.mark_non_differentiable(mean, rstd)
        return y, mean, rstd

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _mean, _rstd):
        need_x, need_scale, need_bias, _ = ctx.needs_input_grad
        dx, dscale, dbias = layer_norm_backward(dy, *ctx.saved_tensors, need_dx=need_x,
                                                need_params=need_scale or need_bias)
        return dx, dscale if need_scale else None, dbias.view(ctx.bias_shape) if need_bias else None, None


class _Dense(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, act, slope, save_pre):
        keep = save_pre or act != "none"
        y, pre = dense(x, w, bias, act, slope, residual, True) if keep else (dense(x, w, bias, act, slope, residual), None)
        ctx.save_for_backward(x, w, None if act == "none" else pre)
        ctx.act, ctx.slope = act, slope
        ctx.bias_shape = None if bias is None else bias.shape
        if keep:
            ctx.mark_non_differentiable(pre)
        return y, pre

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _pre):
        x, w, pre = ctx.saved_tensors
        need_x, need_w, need_bias, need_residual = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_bias:
            try:
                dx, dw, db = dense_backward(dy, x, w, pre, ctx.act, ctx.slope, need_x, need_w, need_bias)
            except _native.MaximError as e:
                # Nobody can poll on autograd's own thread: its records are told by this error.
                if e.code == _native.MX_E_DEVICE:
                    while _native.lib().mx_dense_poll() == _native.MX_E_DEVICE:
                        pass
                raise
        return dx, dw, db.view(ctx.bias_shape) if need_bias else None, dy if need_residual else None, None, None, None


def layer_norm(x, scale, bias, eps=1e-6, stats=False):
    """(x - mean) * rstd * scale + bias over the last dimension. With `stats`
    also the fp32 mean and rstd of every row, which the backward pass takes:
    (y, mean, rstd). scale and bias are of x's type or fp32. Autograd knows of y
    where an input requires a gradient (mean and rstd carry none)."""
    if (x.requires_grad or scale.requires_grad or bias.requires_grad) and torch.is_grad_enabled():
        y, mean, rstd = _LayerNorm.apply(x, scale, bias, eps)
        return (y, mean, rstd) if stats else y
    device, code = _where(x, scale, bias), _dtype(x)
    xp, rows, c, xs, x = _rows(x, "x")
    pt = _param_dtype(scale, x.dtype)
    scale, bias = _vector(scale, pt, c), _vector(bias, pt, c)
    shape = x.shape
    y = _like(x)
    if not stats:
        _launch("mx_layer_norm", _NORM, (xp, scale.data_ptr(), bias.data_ptr(), y.data_ptr(), 0, 0, rows, c, xs, c,
                                         code, _DT[pt], eps, 0), device)
        return y
    # new_empty without a dtype is the quicker call; any fp32 tensor at hand serves.
    f32 = x if x.dtype is torch.float32 else scale
    mean = f32.new_empty(shape[:-1]) if f32.dtype is torch.float32 else x.new_empty(shape[:-1], dtype=torch.float32)
    rstd = torch.empty_like(mean)
    _launch("mx_layer_norm", _NORM, (xp, scale.data_ptr(), bias.data_ptr(), y.data_ptr(), mean.data_ptr(),
                                     rstd.data_ptr(), rows, c, xs, c, code, _DT[pt], eps, 0), device)
    return y, mean, rstd


def layer_norm_backward(dy, x, scale, mean, rstd, need_dx=True, need_params=True):
    """The gradients of layer_norm: (dx, dscale, dbias), None where not needed.
    mean and rstd are the forward pass's."""
    device, code = _where(x, dy, scale, mean, rstd), _dtype(x, dy)
    if dy.shape != x.shape:
        raise ValueError("dy has shape %s, x %s" % (tuple(dy.shape), tuple(x.shape)))
    xp, rows, c, xs, x = _rows(x, "x")
    dyp, _, _, dys, dy = _rows(dy, "dy")
    pt = _param_dtype(scale, x.dtype)
    scale = _vector(scale, pt, c)
    mean, rstd = _vector(mean, torch.float32, rows), _vector(rstd, torch.float32, rows)
    dx = _like(x) if need_dx else None
    dscale = dbias = None
    if need_params:
        dscale, dbias = torch.empty_like(scale), torch.empty_like(scale)
    _launch("mx_layer_norm_backward", _NORM_BACKWARD,
            [dyp, xp, scale.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dx.data_ptr() if need_dx else 0,
             dscale.data_ptr() if need_params else 0, dbias.data_ptr() if need_params else 0, 0, 0, rows, c, dys, xs, c,
             code, _DT[pt]], device, 8)
    return dx, dscale, dbias


def dense(x, w, bias=None, act="none", slope=0.2, residual=None, save_pre=False):
    """act(x @ w.T + bias) + residual: x [..., k], w [n, k], bias [n], residual
    [..., n]. act is one of "none", "gelu" (the erf form), "lrelu" (leaky, with
    `slope`), "sigmoid". With `save_pre` also x @ w.T + bias, which the backward
    pass of an activation takes: (y, pre). Autograd knows of y where an input
    requires a gradient (pre carries none)."""
    if ((x.requires_grad or w.requires_grad or bias is not None and bias.requires_grad or
         residual is not None and residual.requires_grad) and torch.is_grad_enabled()):
        y, pre = _Dense.apply(x, w, bias, residual, act, slope, save_pre)
        return (y, pre) if save_pre else y
    device, code = _where(x, w, bias, residual), _dtype(x, w, bias, residual)
    xp, m, k, xs, x = _rows(x, "x")
    if w.dim() != 2:
        raise ValueError("w has %d dimensions, expected 2" % w.dim())
    wp, n, _, ws, w = _rows(w, "w", k)
    shape = x.shape[:-1] + (n,)
    y = x.new_empty(shape)
    pre = torch.empty_like(y) if save_pre else None
    rp = rs = bp = 0
    if residual is not None:
        if residual.shape != shape:
            raise ValueError("residual has shape %s, the product %s" % (tuple(residual.shape), tuple(shape)))
        rp, _, _, rs, residual = _rows(residual, "residual")
    if bias is not None:
        bias = _vector(bias, x.dtype, n)
        bp = bias.data_ptr()
    _launch("mx_dense", _DENSE, [xp, wp, bp, rp, y.data_ptr(), pre.data_ptr() if save_pre else 0, 0, 0, m, k, n, xs,
                                 ws, rs, n, n, code, _act(act), slope, 0], device, 6)
    return (y, pre) if save_pre else y


def dense_backward(dy, x, w, pre=None, act="none", slope=0.2, need_dx=True, need_dw=True, need_db=True):
    """The gradients of dense: (dx, dw, db), None where not needed. pre is the
    forward pass's (with an activation); the residual's gradient is dy."""
    device, code = _where(dy, x, w, pre), _dtype(dy, x, w, pre)
    if dy.shape[:-1] != x.shape[:-1]:
        raise ValueError("dy has shape %s, x %s" % (tuple(dy.shape), tuple(x.shape)))
    dyp, m, n, dys, dy = _rows(dy, "dy")
    xp, _, k, xs, x = _rows(x, "x")
    if w.dim() != 2 or w.shape[0] != n:
        raise ValueError("w has shape %s, dy rows of %d" % (tuple(w.shape), n))
    wp, _, _, ws, w = _rows(w, "w", k)
    pp = ps = 0
    if act != "none":
        if pre is None or pre.shape != dy.shape:
            raise ValueError("the gradient of %s needs pre, of dy's shape" % act)
        pp, _, _, ps, pre = _rows(pre, "pre")
    dx = _like(x) if need_dx else None
    dw = x.new_empty((n, k)) if need_dw else None
    db = x.new_empty((n,)) if need_db else None
    _launch("mx_dense_backward", _DENSE_BACKWARD,
            [dyp, xp, wp, pp, dx.data_ptr() if need_dx else 0, dw.data_ptr() if need_dw else 0,
             db.data_ptr() if need_db else 0, 0, 0, m, k, n, dys, xs, ws, ps, k, k, code, _act(act), slope, 0], device,
            7)
    return dx, dw, db


def release_workspaces():
    """Give the workspaces that the calling thread's calls have kept (up to 32 MB a
    stream) back to torch's allocator. A thread's go with the thread by themselves."""
    _kept.by_stream.clear()


def poll():
    """`mx_dense_poll`: raise if a dense kernel finished so far gave up a wait in
    its pipeline (its output is then not to be used). Does not wait. Every host
    thread is told once; until then its dense calls on that device are refused."""
    _native.check(_native.lib().mx_dense_poll(), "dense")
