"""Train a residual channel MLP - x + W2 gelu(W1 norm(x) + b1) + b2, the block
that the model's layers and most language models are built of - with the
package's operators, then serve it one token at a time.

    python examples/train_mlp.py [--rows 4096] [--channels 256] [--steps 60] [--dtype bf16]

The block learns to imitate a fixed random teacher of the same shape. Forward
and backward are four calls each of `maxim-rs_b200/ops.py`; parameters and
their gradients stay in the compute type, with fp32 master copies in the
optimiser.
"""
import argparse
import importlib
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
ops = importlib.import_module("maxim-rs_b200.ops")

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


class Mlp:
    """The block, its parameters as a dict of tensors."""

    def __init__(self, channels, hidden, dtype, seed, out_gain=1.0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)

        def normal(*shape, std):
            return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

        self.p = {"scale": torch.ones(channels, device="cuda"), "shift": torch.zeros(channels, device="cuda"),
                  "w1": normal(hidden, channels, std=1 / math.sqrt(channels)),
                  "b1": torch.zeros(hidden, dtype=dtype, device="cuda"),
                  "w2": normal(channels, hidden, std=out_gain / math.sqrt(hidden)),
                  "b2": torch.zeros(channels, dtype=dtype, device="cuda")}

    def serve(self, x):
        """The output alone: any number of tokens, a single one included."""
        p = self.p
        h = ops.dense(ops.layer_norm(x, p["scale"], p["shift"]), p["w1"], p["b1"], act="gelu")
        return ops.dense(h, p["w2"], p["b2"], residual=x)

    def forward(self, x):
        """The output, and what the backward pass reads."""
        p = self.p
        n, mean, rstd = ops.layer_norm(x, p["scale"], p["shift"], stats=True)
        h, pre = ops.dense(n, p["w1"], p["b1"], act="gelu", save_pre=True)
        return ops.dense(h, p["w2"], p["b2"], residual=x), (x, n, mean, rstd, h, pre)

    def backward(self, dy, saved):
        """The input's gradient and the parameters'."""
        p, g = self.p, {}
        x, n, mean, rstd, h, pre = saved
        dh, g["w2"], g["b2"] = ops.dense_backward(dy, h, p["w2"])
        dn, g["w1"], g["b1"] = ops.dense_backward(dh, n, p["w1"], pre=pre, act="gelu")
        dx, g["scale"], g["shift"] = ops.layer_norm_backward(dn, x, p["scale"], mean, rstd)
        return dx + dy, g  # the residual passes dy on


class Adam:
    """Adam over fp32 master copies of a dict of parameters."""

    def __init__(self, params, lr):
        self.params, self.lr, self.t = params, lr, 0
        self.master = {k: v.float().clone() for k, v in params.items()}
        self.m = {k: torch.zeros_like(v) for k, v in self.master.items()}
        self.v = {k: torch.zeros_like(v) for k, v in self.master.items()}

    def step(self, grads):
        self.t += 1
        for k, g in grads.items():
            g = g.float()
            self.m[k].lerp_(g, 0.1)
            self.v[k].lerp_(g * g, 0.01)
            m, v = self.m[k] / (1 - 0.9 ** self.t), self.v[k] / (1 - 0.99 ** self.t)
            self.master[k] -= self.lr * m / (v.sqrt() + 1e-8)
            self.params[k].copy_(self.master[k])


def train(rows, channels, steps, dtype, lr=2e-3, seed=0, report=None):
    """Returns the trained block, its last input and the loss of every step."""
    teacher = Mlp(channels, 4 * channels, dtype, seed + 1)
    student = Mlp(channels, 4 * channels, dtype, seed + 2, out_gain=0.1)
    optimiser = Adam(student.p, lr)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    losses = []
    for step in range(steps):
        x = torch.randn(rows, channels, generator=g, device="cuda").to(dtype)
        y, saved = student.forward(x)
        err = y.float() - teacher.serve(x).float()
        losses.append((err * err).mean())
        _, grads = student.backward((err * (2 / rows)).to(dtype), saved)
        optimiser.step(grads)
        if report and (step % 10 == 0 or step == steps - 1):
            report(step, losses[-1].item())
    ops.poll()
    return student, x, [v.item() for v in losses]


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--rows", type=int, default=4096)
    ap.add_argument("--channels", type=int, default=256)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--dtype", choices=sorted(DTYPES), default="bf16")
    a = ap.parse_args()
    block, x, losses = train(a.rows, a.channels, a.steps, DTYPES[a.dtype],
                             report=lambda s, v: print("step %3d  loss %.5f" % (s, v)))
    whole = block.serve(x)
    one = torch.cat([block.serve(x[i:i + 1]) for i in range(8)])
    print("served token by token: largest difference %.3g" % (one.float() - whole[:8].float()).abs().max().item())
    return 0 if losses[-1] < losses[0] else 1


if __name__ == "__main__":
    sys.exit(main())
