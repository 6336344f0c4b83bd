#!/usr/bin/env python3
"""A stack of gated feed-forward blocks, trained and then run token by token.

Each block is ``branch = GatedMLP(n)`` followed by ``ResidualNorm``: the norm of
the branch, dropout, the residual sum and the norm before the next block in one
pass.  The weights are trained in bfloat16 with Float32 master copies (AdamW)
until the stack reproduces fixed random targets on a fixed batch; then single
tokens go through the few-row kernels, in a captured graph, and give the
batch's rows.

    python examples/feed_forward.py [--layers 2] [--dim 256] [--hidden 704] [--tokens 256]
                                    [--steps 60] [--p 0.05] [--dtype bf16|f32]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import momijo_amd as mj  # noqa: E402


class Stack:
    """Layers of (GatedMLP, ResidualNorm) after one norm; its output is the last norm's."""

    def __init__(self, layers: int, dim: int, hidden: int, p: float, dtype, seed: int = 0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda r, c: torch.randn((r, c), generator=gen, device="cuda") * c ** -0.5  # noqa: E731
        self.dtype = dtype
        self.masters, self.mlps = [], []
        for _ in range(layers):
            w = [normal(hidden, dim), normal(hidden, dim), normal(dim, hidden)]
            self.masters.append(w)
            self.mlps.append(mj.GatedMLP(*(t.to(dtype) for t in w)))
        self.first = torch.ones(dim, device="cuda")
        # a seed of its own for every layer: equal seeds would drop the same places
        self.norms = [mj.ResidualNorm(dim, p=p, seed=seed * layers + i) for i in range(layers)]

    def parameters(self):
        out = [self.first]
        for w, norm in zip(self.masters, self.norms):
            out += w + [norm.post_weight, norm.next_weight]
        return out

    def refresh(self):
        """The working weights from the masters, in place (a captured graph sees them)."""
        for w, mlp in zip(self.masters, self.mlps):
            for t, m in zip((mlp.gate, mlp.up, mlp.down), w):
                t.copy_(m)

    def forward(self, x):
        y, n = mj.residual_norm(x, next_weight=self.first)
        for mlp, norm in zip(self.mlps, self.norms):
            y, n = norm.forward(y, mlp.forward(n))
        return n

    def forward_train(self, x):
        y, n, start = mj.residual_norm_train(x, next_weight=self.first)
        saved = []
        for mlp, norm in zip(self.mlps, self.norms):
            b, s = mlp.forward_train(n)
            y, n, t = norm.forward_train(y, b)
            saved.append((s, t))
        return n, (start, saved)

    def backward(self, dn, state):
        """Gradients in the order of parameters()."""
        start, saved = state
        dy, grads = None, []
        for mlp, norm, (s, t) in reversed(list(zip(self.mlps, self.norms, saved))):
            g = norm.backward(dy, dn, t)
            dy = g["x"]
            dn, *dw = mlp.backward(g["branch"], s)
            grads.append(dw + [g["post_weight"], g["next_weight"]])
        first = mj.residual_norm_backward(dy, dn, start)["next_weight"]
        return [first] + [t for layer in reversed(grads) for t in layer]


def train(stack: Stack, x, target, steps: int, lr: float = 2e-3):
    """The mean squared error before each step."""
    params = stack.parameters()
    opt = torch.optim.AdamW(params, lr=lr, weight_decay=0.0)
    losses = []
    for _ in range(steps):
        n, state = stack.forward_train(x)
        diff = n.float() - target
        losses.append(diff.square().mean())
        dn = (diff * (2.0 / diff.numel())).to(stack.dtype)
        for p, g in zip(params, stack.backward(dn, state)):
            p.grad = g.float()
        opt.step()
        stack.refresh()
    return [float(v) for v in losses]


def decoder(stack: Stack, dim: int):
    """A captured one-token pass: call it with a row, get the output row."""
    x = torch.zeros((1, dim), dtype=stack.dtype, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        stack.forward(x)
        side.synchronize()
        graph.capture_begin()
        out = stack.forward(x)
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(side)

    def step(row):
        x.copy_(row.reshape(1, dim))
        graph.replay()
        return out.clone()

    return step


def main(argv=None):
    a = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    a.add_argument("--layers", type=int, default=2)
    a.add_argument("--dim", type=int, default=256)
    a.add_argument("--hidden", type=int, default=704)
    a.add_argument("--tokens", type=int, default=256)
    a.add_argument("--steps", type=int, default=60)
    a.add_argument("--p", type=float, default=0.05)
    a.add_argument("--dtype", choices=("bf16", "f32"), default="bf16")
    a = a.parse_args(argv)
    dtype = torch.bfloat16 if a.dtype == "bf16" else torch.float32
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((a.tokens, a.dim), generator=gen, device="cuda").to(dtype)
    target = torch.randn((a.tokens, a.dim), generator=gen, device="cuda")
    stack = Stack(a.layers, a.dim, a.hidden, a.p, dtype)
    losses = train(stack, x, target, a.steps)
    whole = stack.forward(x)
    step = decoder(stack, a.dim)
    rows = torch.cat([step(x[i]) for i in range(min(8, a.tokens))])
    worst = float((rows.float() - whole[:rows.shape[0]].float()).abs().max())
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps; one-token rows differ from "
          f"the batch's by at most {worst:.2e}")
    return losses, worst


if __name__ == "__main__":
    main()
