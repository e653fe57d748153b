"""An MoE layer on one MI355X: training steps and a decoding step, from router logits to the residual stream.

    python examples/moe_layer.py [--tokens 8192] [--experts 32] [--top-k 4] [--hidden 2880] [--inner 2880] [--steps 5]

The router is a plain torch product; everything behind it is the package's: routing, dispatch, the experts' FP8
products with bias and gated activation, and the combination, forward and backward. Weights and tokens are random.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from __graft_entry__ import load_package  # noqa: E402

ggemm = load_package()


class MoE(torch.nn.Module):
    def __init__(self, hidden, inner, experts, top_k):
        super().__init__()
        make = lambda *s: torch.nn.Parameter(torch.randn(s, device="cuda", dtype=torch.bfloat16) * 0.02)  # noqa: E731
        self.router, self.top_k = make(experts, hidden), top_k
        self.w_up, self.b_up = make(experts, 2 * inner, hidden), make(experts, 2 * inner)
        self.w_down, self.b_down = make(experts, hidden, inner), make(experts, hidden)
        self.caches = (ggemm.FP8WeightCache(), ggemm.FP8WeightCache())

    def forward(self, x):
        logits = x @ self.router.t()
        return ggemm.moe_layer_fp8(x, logits, self.w_up, self.w_down, self.top_k, bias_up=self.b_up,
                                   bias_down=self.b_down, slope=1.702, limit=7.0, shift=1.0, residual=x,
                                   weight_caches=self.caches)


def timed(f, n):
    f()
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(n):
        r = f()
    torch.cuda.synchronize()
    return r, (time.perf_counter() - t) / n * 1e3


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("tokens", 8192), ("experts", 32), ("top-k", 4), ("hidden", 2880), ("inner", 2880), ("steps", 5)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    torch.manual_seed(0)
    layer = MoE(a.hidden, a.inner, a.experts, a.top_k)
    opt = torch.optim.SGD(layer.parameters(), lr=1e-2)
    for c in layer.caches:
        c.attach(opt)
    x = torch.randn((a.tokens, a.hidden), device="cuda", dtype=torch.bfloat16)
    target = torch.randn_like(x)

    def step():
        opt.zero_grad(set_to_none=True)
        loss = torch.nn.functional.mse_loss(layer(x).float(), target.float())
        loss.backward()
        opt.step()
        return loss

    losses, ms = [], 0.0
    for _ in range(a.steps):
        loss, ms = timed(step, 1)
        losses.append(float(loss.detach()))
    print(f"training: {a.tokens} tokens, {a.experts} experts of {a.hidden} x {a.inner}, top {a.top_k}: {ms:.2f} ms a step, "
          f"loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    with torch.no_grad():
        one = x[:1]
        _, ms = timed(lambda: layer(one), 50)
        print(f"decoding: 1 token, {ms * 1e3:.0f} us")
    return losses


if __name__ == "__main__":
    main()
