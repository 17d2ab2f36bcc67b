"""Trains a small residual network with the layer products and AdamW, and serves it one token at a time.

Two blocks  h = gelu_tanh(x W1^T + b1),  x + h W2^T + b2  in BF16 learn a fixed random map of the same form; AdamW keeps
32-bit master weights and 8-bit moments. The product of one layer is then compared with the library's FP64 product of
the same values, and the trained network answers single tokens, whose rows must be those of the batch.

    python examples/train_mlp.py [--steps 200] [--width 512] [--tokens 2048]
"""

import argparse
import math
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import oztt_b200 as oz


def weights(width, blocks, generator):
    """W1 [4 width, width], b1, W2 [width, 4 width], b2 of every block."""
    def normal(*shape, scale):
        return (scale * torch.randn(*shape, device="cuda", generator=generator)).to(torch.bfloat16)

    return [(normal(4 * width, width, scale=1 / math.sqrt(width)), normal(4 * width, scale=0.1),
             normal(width, 4 * width, scale=0.5 / math.sqrt(width)), normal(width, scale=0.1)) for _ in range(blocks)]


def forward(x, blocks, keep=None):
    """The network's output; keep receives what the backward pass needs."""
    for w1, b1, w2, b2 in blocks:
        if keep is None:
            h = oz.linear(x, w1, b1, activation="gelu_tanh")
        else:
            h, pre = oz.linear(x, w1, b1, activation="gelu_tanh", save_pre=True)
            keep.append((x, h, pre))
        x = oz.linear(h, w2, b2, residual=x)
    return x


def backward(dy, blocks, keep):
    """The gradients of all weights, in the order of the optimiser's list."""
    grads = []
    for (w1, b1, w2, b2), (x, h, pre) in zip(reversed(blocks), reversed(keep)):
        dh, dw2, db2 = oz.linear_backward(dy, h, w2)
        dx, dw1, db1 = oz.linear_backward(dh, x, w1, pre=pre, activation="gelu_tanh")
        grads = [dw1, db1, dw2, db2] + grads
        dy = dy + dx  # the residual's gradient is dy itself
    return grads


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--width", type=int, default=512)
    ap.add_argument("--tokens", type=int, default=2048)
    a = ap.parse_args()
    gen = torch.Generator(device="cuda").manual_seed(0)
    teacher, student = weights(a.width, 2, gen), weights(a.width, 2, gen)
    params = [p for block in student for p in block]
    opt = oz.AdamW(params, lr=2e-3, betas=(0.9, 0.95), weight_decay=0.0, masters=True, state_bits=8)

    losses = []
    for step in range(a.steps):
        x = torch.randn(a.tokens, a.width, device="cuda", generator=gen).to(torch.bfloat16)
        keep = []
        error = forward(x, student, keep).float() - forward(x, teacher).float()
        losses.append((error * error).mean())
        grads = backward((error * (2 / error.numel() * 1024)).to(torch.bfloat16), student, keep)
        norm = torch.sqrt(sum((g.float() ** 2).sum() for g in grads)) / 1024  # (the loss was scaled by 1024)
        opt.step(grads, grad_scale=(torch.clamp(1.0 / norm, max=1.0) / 1024).reshape(1),
                 lr=2e-3 * min(1.0, (step + 1) / 20) * (1 - step / a.steps))
        if step % 50 == 0 or step == a.steps - 1:
            print(f"step {step:4d}  mean squared error {float(losses[-1]):.5f}")

    # one product against the library's FP64 product of the same values
    w1 = student[0][0]
    z = oz.linear(x[:128], w1).double().cpu().numpy()
    a64, b64 = x[:128].double().cpu().numpy(), w1.t().double().cpu().numpy()
    ref = oz.Context().multiply(a64, b64, 128, w1.shape[0], a.width, oz.Options(format=oz.Format.INT8)).reshape(z.shape)
    off = np.abs(z - ref).max() / np.abs(ref).max()
    print(f"BF16 product against the FP64 product: {off:.2e} of the largest value")

    # serving: a token at a time
    batch = forward(x[:64], student).float()
    single = torch.cat([forward(x[i:i + 1], student) for i in range(64)]).float()
    apart = float((batch - single).abs().max() / batch.abs().max())
    print(f"64 single tokens against the batch: {apart:.2e} of the largest value")
    assert float(losses[-1]) < 0.5 * float(losses[0]) and off < 2 ** -8 and apart < 2 ** -6
    print("ok")


if __name__ == "__main__":
    main()
