"""A gated feed-forward block: trained in 16 bits for some steps, then served with weights in 8-bit integers.

    python examples/feed_forward.py [--dtype bf16] [--act silu] [--steps 8]

One block with random weights.  Training takes `cmpext3.gated_linear` and its gradients for the first half (the
second projection is torch's own here); serving quantises the trained weights once and takes a prompt and then
single tokens through `int8_gated_linear` and `int8_linear`.  The script prints the times and how far the served
block is from the trained one.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import cmpext3  # noqa: E402


class FeedForward:
    """y = (act(x Wg^T) * (x Wu^T)) Wd^T; both halves of the first projection are one tensor."""

    def __init__(self, width, inner, act, dtype, device, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
        self.inner, self.act = inner, act
        self.w_in = (rand(2 * inner, width) * width**-0.5).to(dtype).requires_grad_()
        self.w_down = (rand(width, inner) * inner**-0.5).to(dtype).requires_grad_()

    def forward(self, x):
        h = cmpext3.gated_linear(x, self.w_in[: self.inner], self.w_in[self.inner :], self.act)
        return torch.nn.functional.linear(h, self.w_down)


class ServedFeedForward:
    """The same block with its weights in codes, a scale for each row of a weight."""

    def __init__(self, block):
        with torch.no_grad():
            codes, self.scale = cmpext3.quantize_int8(block.w_in)
            self.w_down, self.down_scale = cmpext3.quantize_int8(block.w_down)
        n = block.inner
        self.gate, self.up, self.gate_scale, self.up_scale = codes[:n], codes[n:], self.scale[:n], self.scale[n:]
        self.act = block.act

    def forward(self, x):
        h = cmpext3.int8_gated_linear(x, self.gate, self.up, self.gate_scale, self.up_scale, self.act)
        return cmpext3.int8_linear(h, self.w_down, self.down_scale)


def train_step(block, x, target, rate):
    """One step of plain gradient descent; returns the loss (a tensor: nothing waits for the GPU)."""
    loss = (block.forward(x).float() - target).square().mean()
    weights = (block.w_in, block.w_down)
    with torch.no_grad():
        for w, g in zip(weights, torch.autograd.grad(loss, weights)):
            w -= rate * g
    return loss.detach()


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--dtype", choices=["fp16", "bf16"], default="bf16")
    ap.add_argument("--act", choices=["silu", "gelu", "gelu_tanh", "relu"], default="silu")
    ap.add_argument("--width", type=int, default=1024)
    ap.add_argument("--inner", type=int, default=2816)
    ap.add_argument("--tokens", type=int, default=512)
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args()
    dtype = {"fp16": torch.float16, "bf16": torch.bfloat16}[a.dtype]
    block = FeedForward(a.width, a.inner, a.act, dtype, "cuda")
    x = torch.randn(a.tokens, a.width, device="cuda").to(dtype)
    target = torch.randn(a.tokens, a.width, device="cuda")

    def timed(what, n, f):
        f()
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(n):
            out = f()
        torch.cuda.synchronize()
        print(f"{what}: {1e6 * (time.perf_counter() - t) / n:.1f} us")
        return out

    if a.steps:
        loss = timed(f"training step of {a.tokens} tokens", a.steps, lambda: train_step(block, x, target, 0.5))
        print(f"loss {loss.item():.4f}")
    served = ServedFeedForward(block)
    with torch.no_grad():
        for tokens in (a.tokens, 1):
            y = timed(f"{tokens} tokens in 16 bits", 20, lambda: block.forward(x[:tokens]))
            z = timed(f"{tokens} tokens in 8-bit integers", 20, lambda: served.forward(x[:tokens]))
            print(f"relative difference {((y.float() - z.float()).norm() / y.float().norm()).item():.2e}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
