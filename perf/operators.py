"""Cases that measure the training and serving operators on the caller's own
device tensors: layer norm and the dense product (bias, activation and residual
in its epilogue), each forward and backward.

With `own` false a pass runs the operator in plain torch operations in 32
bits, rounded once at the end; with `own` true it makes the calls a user makes
(`maxim-rs_b200/ops.py`). `exact` computes the same outputs from the
definitions in 64 bits.
"""
import importlib
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6  # the framework's layer norm
SLOPE = 0.2  # its leaky ReLU

# The largest listed sizes, which bound the drawn ones.
MAX_LN_VALUES = 16411 * 4096
MAX_DENSE_MACS = 8192 * 4096 * 8192
MAX_DENSE_VALUES = 1146880 * 64


def listed():
    return [
        # One token of a decoding step before its projection: launch latency.
        {"name": "ln_token_bf16", "op": "ln", "rows": 1, "c": 4096, "dtype": "bf16", "param": "f32"},
        # The image model's own norm at half resolution (448x640, 64 channels).
        {"name": "ln_pixels_f32", "op": "ln", "rows": 448 * 640, "c": 64, "dtype": "f32", "param": "f32"},
        # A training batch of tokens, a row count that no tile divides.
        {"name": "ln_tokens_bf16", "op": "ln", "rows": 16411, "c": 4096, "dtype": "bf16", "param": "f32"},
        # Backward of one short sequence, odd width: rows that are not 16-byte aligned.
        {"name": "ln_grad_odd_f16", "op": "ln_grad", "rows": 77, "c": 769, "dtype": "f16", "param": "f16"},
        # Backward of the image model's full-resolution norm: very many short rows
        # whose parameter gradients are sums over all of them.
        {"name": "ln_grad_pixels_f32", "op": "ln_grad", "rows": 896 * 1280, "c": 32, "dtype": "f32", "param": "f32"},
        # Backward of the training batch of tokens.
        {"name": "ln_grad_tokens_bf16", "op": "ln_grad", "rows": 16411, "c": 4096, "dtype": "bf16", "param": "f32"},
        # One token through a widening layer: the weights' bytes alone count.
        {"name": "dense_token_bf16", "op": "dense", "m": 1, "k": 4096, "n": 16384, "dtype": "bf16", "act": "gelu",
         "residual": False, "pre": False},
        # A short prompt at odd sizes with a residual: unaligned rows, few tiles.
        {"name": "dense_odd_f16", "op": "dense", "m": 517, "k": 1023, "n": 771, "dtype": "f16", "act": "lrelu",
         "residual": True, "pre": False},
        # The image model's widening 1x1 product at quarter resolution (224x320), in
        # full precision, keeping what its backward pass needs.
        {"name": "dense_pixels_f32", "op": "dense", "m": 224 * 320, "k": 128, "n": 256, "dtype": "f32",
         "act": "gelu", "residual": False, "pre": True},
        # A training batch through a widening layer.
        {"name": "dense_tokens_bf16", "op": "dense", "m": 8192, "k": 4096, "n": 8192, "dtype": "bf16", "act": "gelu",
         "residual": False, "pre": True},
        # Backward of the image model's product: a long sum over pixels into a small matrix.
        {"name": "dense_grad_pixels_f32", "op": "dense_grad", "m": 224 * 320, "k": 128, "n": 256, "dtype": "f32",
         "act": "gelu"},
        # Backward of a training batch through a square layer.
        {"name": "dense_grad_tokens_bf16", "op": "dense_grad", "m": 8192, "k": 4096, "n": 4096, "dtype": "bf16",
         "act": "gelu"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width over [lo, hi]: as it falls (odd ones among them), or rounded to a
    multiple of 8 or 64, as most models' widths are."""
    v = _log_int(rng, lo, hi)
    q = rng.choice([1, 8, 64, 64])
    return max(lo, v - v % q) if v >= q else v


def draw(rng):
    op = rng.choice(["ln", "ln_grad", "dense", "dense_grad"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op in ("ln", "ln_grad"):
        c = _width(rng, 3, 16384)
        limit = MAX_LN_VALUES // (2 if dtype == "f32" else 1)
        rows = _log_int(rng, 1, min(1146880, limit // c))
        param = rng.choice([dtype, "f32"])
        return {"op": op, "rows": rows, "c": c, "dtype": dtype, "param": param}
    k = _width(rng, 3, 8192)
    n = _width(rng, 3, 16384)
    # A product in full precision is three in the tensor cores' terms, and the
    # backward pass is two.
    macs = MAX_DENSE_MACS // ((4 if dtype == "f32" else 1) * (2 if op == "dense_grad" else 1))
    values = MAX_DENSE_VALUES // (2 if dtype == "f32" else 1)
    m = _log_int(rng, 1, max(1, min(1146880, macs // (k * n), values // max(k, n))))
    act = rng.choice(["none", "gelu", "lrelu", "sigmoid"])
    case = {"op": op, "m": m, "k": k, "n": n, "dtype": dtype, "act": act}
    if op == "dense":
        case["residual"] = rng.random() < 0.5
        case["pre"] = act != "none" and rng.random() < 0.5
    return case


def _inputs(case, seed):
    """The tensors of a case, made on the GPU from the seed."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    dt = DTYPES[case["dtype"]]
    if case["op"] in ("ln", "ln_grad"):
        rows, c = case["rows"], case["c"]
        pt = DTYPES[case["param"]]
        # A residual stream: channels of unequal spread about a common offset.
        spread = torch.exp(0.5 * normal(c))
        x = normal(rows, c).mul_(spread).add_(0.3).to(dt)
        t = {"x": x, "scale": (1.0 + 0.1 * normal(c)).to(pt), "bias": (0.1 * normal(c)).to(pt)}
        if case["op"] == "ln_grad":
            t["dy"] = normal(rows, c).to(dt)
            xf = x.float()
            mean = xf.sum(1) / c
            xf.sub_(mean[:, None])
            t["mean"] = mean
            t["rstd"] = 1.0 / torch.sqrt((xf * xf).sum(1) / c + EPS)
        return t
    m, k, n = case["m"], case["k"], case["n"]
    t = {"x": normal(m, k).to(dt), "w": (normal(n, k) / math.sqrt(k)).to(dt)}
    if case["op"] == "dense":
        t["bias"] = (0.1 * normal(n)).to(dt)
        if case["residual"]:
            t["residual"] = normal(m, n).to(dt)
    else:
        t["dy"] = normal(m, n).to(dt)
        if case["act"] != "none":
            t["pre"] = normal(m, n).to(dt)
    return t


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:
        state["ops"] = importlib.import_module("maxim-rs_b200.ops")
    return state


def _act(v, act):
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * 0.7071067811865476))
    if act == "lrelu":
        return torch.where(v >= 0, v, SLOPE * v)
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-v))
    return v


def _act_grad(v, act):
    if act == "gelu":
        phi = torch.exp(-0.5 * v * v) * 0.3989422804014327
        return 0.5 * (1.0 + torch.erf(v * 0.7071067811865476)) + v * phi
    if act == "lrelu":
        return torch.where(v >= 0, 1.0, SLOPE)
    s = 1.0 / (1.0 + torch.exp(-v))
    return s * (1.0 - s)


def _plain(state):
    case = state["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    x = state["x"].float()
    if op == "ln":
        c = case["c"]
        mean = x.sum(1) / c
        d = x - mean[:, None]
        rstd = 1.0 / torch.sqrt((d * d).sum(1) / c + EPS)
        y = d * rstd[:, None] * state["scale"].float() + state["bias"].float()
        return y.to(dt), mean, rstd
    dyf = state["dy"].float() if "dy" in state else None
    if op == "ln_grad":
        c, pt = case["c"], DTYPES[case["param"]]
        rstd = state["rstd"][:, None]
        xhat = (x - state["mean"][:, None]) * rstd
        dscale = (dyf * xhat).sum(0)
        dbias = dyf.sum(0)
        gr = dyf * state["scale"].float()
        dx = rstd * (gr - gr.sum(1, keepdim=True) / c - xhat * ((gr * xhat).sum(1, keepdim=True) / c))
        return dx.to(dt), dscale.to(pt), dbias.to(pt)
    w = state["w"].float()
    if op == "dense":
        pre = x @ w.t() + state["bias"].float()
        y = _act(pre, case["act"])
        if case["residual"]:
            y = y + state["residual"].float()
        return (y.to(dt), pre.to(dt)) if case["pre"] else y.to(dt)
    if case["act"] != "none":
        dyf = dyf * _act_grad(state["pre"].float(), case["act"])
    return (dyf @ w).to(dt), (dyf.t() @ x).to(dt), dyf.sum(0).to(dt)


def run(state):
    if not own:
        return _plain(state)
    ops, case = state["ops"], state["case"]
    if case["op"] == "ln":
        return ops.layer_norm(state["x"], state["scale"], state["bias"], eps=EPS, stats=True)
    if case["op"] == "ln_grad":
        return ops.layer_norm_backward(state["dy"], state["x"], state["scale"], state["mean"], state["rstd"])
    if case["op"] == "dense":
        return ops.dense(state["x"], state["w"], state["bias"], act=case["act"], slope=SLOPE,
                         residual=state.get("residual"), save_pre=case["pre"])
    return ops.dense_backward(state["dy"], state["x"], state["w"], pre=state.get("pre"), act=case["act"], slope=SLOPE)


def exact(case, seed):
    """The outputs in 64 bits: statistics by torch's own reductions of doubles,
    the activations' derivatives by differentiating the activation."""
    t = {k: v.double() for k, v in _inputs(case, seed).items()}
    if case["op"] == "ln":
        var, mean = torch.var_mean(t["x"], dim=1, correction=0)
        rstd = torch.rsqrt(var + EPS)
        y = torch.addcmul(t["bias"], (t["x"] - mean.unsqueeze(1)) * rstd.unsqueeze(1), t["scale"])
        return y, mean, rstd
    if case["op"] == "ln_grad":
        # y_j = scale_j n_j + bias_j with n = (x - mean) rstd: the gradient of n
        # projected off the constant vector and off n itself.
        n = (t["x"] - t["mean"].unsqueeze(1)) * t["rstd"].unsqueeze(1)
        gn = t["dy"] * t["scale"]
        along = torch.einsum("rc,rc->r", gn, n) / case["c"]
        dx = t["rstd"].unsqueeze(1) * (gn - gn.mean(1, keepdim=True) - along.unsqueeze(1) * n)
        return dx, torch.einsum("rc,rc->c", t["dy"], n), t["dy"].sum(0)

    def activation(v):
        if case["act"] == "gelu":
            return v * torch.special.ndtr(v)
        if case["act"] == "lrelu":
            return v.clamp(min=0) + SLOPE * v.clamp(max=0)
        if case["act"] == "sigmoid":
            return torch.sigmoid(v)
        return v

    if case["op"] == "dense":
        pre = torch.addmm(t["bias"], t["x"], t["w"].t())
        y = activation(pre)
        if case["residual"]:
            y = y + t["residual"]
        return (y, pre) if case["pre"] else y
    d = t["dy"]
    if case["act"] == "lrelu":
        d = torch.where(t["pre"] < 0, SLOPE * d, d)
    elif case["act"] != "none":
        pre = t["pre"].requires_grad_(True)
        with torch.enable_grad():
            (d,) = torch.autograd.grad(activation(pre), pre, d)
    return torch.mm(d, t["w"]), torch.mm(d.t(), t["x"]), d.sum(0)


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("ln", "ln_grad"):
        rows, c = case["rows"], case["c"]
        pe = 4 if case["param"] == "f32" else 2
        if case["op"] == "ln":
            return {"bytes": 2 * rows * c * e + 8 * rows + 2 * c * pe, "flops": 8 * rows * c}
        return {"bytes": 3 * rows * c * e + 8 * rows + 3 * c * pe, "flops": 14 * rows * c}
    m, k, n = case["m"], case["k"], case["n"]
    if case["op"] == "dense":
        outs = 1 + case["pre"] + case["residual"]
        return {"bytes": e * (m * k + n * k + n + outs * m * n), "flops": 2 * m * n * k}
    ins = 1 + (case["act"] != "none")
    return {"bytes": e * (2 * m * k + 2 * n * k + n + ins * m * n), "flops": 4 * m * n * k}
