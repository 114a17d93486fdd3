"""A gated feed-forward block from training in 16 bits to serving in 4.

Trains y = (act(x Wg^T) * (x Wu^T)) Wd^T towards a random teacher block with `gated_linear` and
`gated_linear_backward` (f32 master weights, bf16 copies for the kernels, Adam), then quantises the trained weights
to MXFP4 once and serves it with `gated_linear_mxfp4` and `linear_mxfp4`, for a batch and for single tokens.

    python examples/gated_block.py [--dim 384] [--ffn 1536] [--tokens 2048] [--steps 60]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from tenzor_b200 import ops  # noqa: E402
from tenzor_b200.runtime import Context  # noqa: E402


def block(ctx, x, wg, wu, wd, act):
    h = ops.gated_linear(ctx, x, wg, wu, act)
    return h, h @ wd.t()


def train(ctx, dim, ffn, tokens, steps, act="silu", lr=2e-3, seed=0):
    """Returns the trained bf16 weights (wg, wu, wd) and the loss of every step."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape, std):
        return torch.randn(shape, generator=gen, device="cuda") * std

    shapes = [(ffn, dim), (ffn, dim), (dim, ffn)]
    teacher = [rand(*s, std=s[1] ** -0.5).bfloat16() for s in shapes]
    master = [t.float() + rand(*s, std=0.5 * s[1] ** -0.5) for t, s in zip(teacher, shapes)]
    opt = torch.optim.Adam(master, lr=lr)
    losses = []
    for _ in range(steps):
        x = rand(tokens, dim, std=1.0).bfloat16()
        target = block(ctx, x, *teacher, act)[1]
        wg, wu, wd = (w.bfloat16() for w in master)
        h, y = block(ctx, x, wg, wu, wd, act)
        diff = y.float() - target.float()
        losses.append(diff.square().mean())
        dy = (diff * (2.0 / dim)).bfloat16()  # per-token mean over the outputs; the mean over tokens goes to Adam
        dx, dwg, dwu = ops.gated_linear_backward(ctx, x, wg, wu, dy @ wd, act)
        for w, g in zip(master, (dwg, dwu, dy.t() @ h)):
            w.grad = g.float() / tokens
        opt.step()
    return [w.bfloat16() for w in master], [float(v) for v in losses]


class ServedBlock:
    """The block in MXFP4: weights quantised once, x and h quantised in each call."""

    def __init__(self, ctx, wg, wu, wd, act="silu"):
        self.ctx, self.act = ctx, act
        self.w_in = ops.pack_gated_mxfp4(ctx, wg, wu)
        self.w_out = ops.quantize_mxfp4(ctx, wd)

    def __call__(self, x):
        return ops.linear_mxfp4(self.ctx, ops.gated_linear_mxfp4(self.ctx, x, self.w_in, self.act), self.w_out)


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--dim", type=int, default=384)
    ap.add_argument("--ffn", type=int, default=1536)
    ap.add_argument("--tokens", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=60)
    a = ap.parse_args(argv)
    ctx = Context(0)
    weights, losses = train(ctx, a.dim, a.ffn, a.tokens, a.steps)
    served = ServedBlock(ctx, *weights)
    x = torch.randn(a.tokens, a.dim, device="cuda").bfloat16()
    y16, y4 = block(ctx, x, *weights, "silu")[1].float(), served(x).float()
    cos = torch.nn.functional.cosine_similarity(y16, y4, dim=1)
    one = torch.cat([served(x[i:i + 1]) for i in range(4)]).float()
    same = float((one - y4[:4]).abs().max() / y4[:4].abs().max())
    ctx.check_status()
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps; 4-bit against 16-bit output: cosine "
          f"{float(cos.mean()):.4f} (lowest {float(cos.min()):.4f}); one token against the batch: {same:.1e}")
    return losses, cos, same


if __name__ == "__main__":
    main()
