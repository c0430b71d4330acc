"""What a backward pass costs on the host before any kernel: torch.autograd.grad of a node that launches nothing (the backward of `cat` hands out
views) with 1 .. 8 gradients, next to the backward of the norms around a residual block on rows so few that the GPU waits for the host.

    python tools/autograd_cost.py
"""
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from fluidnet_amd.models.block_norm import gated_residual  # noqa: E402


def us(f, n=2000):
    best = float("inf")
    for _ in range(5):
        for _ in range(20):
            f()
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(n):
            f()
        torch.cuda.synchronize()
        best = min(best, (time.perf_counter() - t) / n * 1e6)
    return best


def main():
    print("us a pass, wall clock, best of 5 times 2000")
    for k in (1, 3, 8):
        parts = [torch.zeros(64, device="cuda", requires_grad=True) for _ in range(k)]
        whole, up = torch.cat(parts), torch.ones(64 * k, device="cuda")
        print(f"cat, {k} gradients (views, no kernel): {us(lambda: torch.autograd.grad(whole, parts, up, retain_graph=True)):.1f}")
    N, C = 16, 256
    x, branch, gate, up = (torch.randn(N, C, device="cuda") for _ in range(4))
    vectors = [torch.rand(C, device="cuda") for _ in range(5)]
    with torch.no_grad():
        print(f"gated_residual forward alone: {us(lambda: gated_residual(x, branch, gate, post_weight=vectors[0], pre_weight=vectors[1])):.1f}")
    for k in (1, 2, 3, 8):
        leaves = [t.clone().requires_grad_(i < k) for i, t in enumerate((x, branch, gate, *vectors))]
        X, B, G, S, W1, B1, W2, B2 = leaves
        y, h = gated_residual(X, B, G, S, post_weight=W1, post_bias=B1, pre_weight=W2, pre_bias=B2, kind="layer", gate_act="sigmoid")
        t = us(lambda: torch.autograd.grad((y, h), leaves[:k], (up, up), retain_graph=True))
        print(f"gated_residual backward, {k} gradients, {2 if k > 3 else 1} launch(es): {t:.1f}")


if __name__ == "__main__":
    main()
