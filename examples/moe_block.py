"""A mixture-of-experts block: one training step and a step of serving.

    y = x + combine(relu(dispatch(norm(x)) @ w1[e]) @ w2[e])

``norm`` is a layer norm, every token goes to its ``k`` best experts, and the
experts are the grouped products of ``mojodgl.ops``.  The package has no
automatic differentiation, so the way back is written out: each operator's
gradient next to the operator.

    python examples/moe_block.py [--tokens 8192] [--width 1024] [--hidden 2048] [--experts 32] [--k 4] [--steps 20]
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mojo-dgl_b200"))

from mojodgl import ops  # noqa: E402


class MoEBlock:
    """Parameters in bfloat16 (the norm's, the router's and the balance bias in
    float32); the router scores with a sigmoid and renormalises its weights."""

    def __init__(self, width, hidden, experts, k, seed=0, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)

        def randn(*shape, scale, dtype=torch.bfloat16):
            return (torch.randn(*shape, device=device, generator=g) * scale).to(dtype)

        self.k, self.experts = k, experts
        self.route = {"score": "sigmoid", "renormalize": True}
        self.params = {
            "norm_weight": torch.ones(width, device=device), "norm_bias": torch.zeros(width, device=device),
            "router": randn(width, experts, scale=width ** -0.5, dtype=torch.float32),
            "w1": randn(experts, width, hidden, scale=width ** -0.5),
            "w2": randn(experts, hidden, width, scale=hidden ** -0.5),
        }
        self.balance = torch.zeros(experts, device=device)

    def forward(self, x):
        p = self.params
        h, mean, rstd = ops.layer_norm(x, p["norm_weight"], p["norm_bias"], return_stats=True)
        logits = h.float() @ p["router"]
        weights, indices = ops.route_topk(logits, self.k, bias=self.balance, **self.route)
        plan = ops.expert_plan(indices, self.experts)
        rows = ops.dispatch(h, plan.positions)
        a1 = ops.segment_mm(rows, p["w1"], plan.counts).relu_()
        a2 = ops.segment_mm(a1, p["w2"], plan.counts)
        y = x + ops.combine(a2, plan.positions, weights)
        return y, (x, h, mean, rstd, logits, weights, indices, plan, rows, a1, a2)

    def backward(self, dy, saved):
        """Gradients of the input and of every parameter."""
        p = self.params
        x, h, mean, rstd, logits, weights, indices, plan, rows, a1, a2 = saved
        da2, dweights = ops.combine_backward(dy, a2, plan.positions, weights)
        da1, dw2 = ops.segment_mm_backward(da2, a1, p["w2"], plan.counts)
        da1.masked_fill_(a1 <= 0, 0)
        drows, dw1 = ops.segment_mm_backward(da1, rows, p["w1"], plan.counts)
        dlogits = ops.route_topk_backward(dweights, logits, indices, **self.route)
        dh = ops.combine(drows, plan.positions).float() + dlogits @ p["router"].T
        dx, dnw, dnb = ops.layer_norm_backward(dh.to(x.dtype), x, mean, rstd, p["norm_weight"])
        grads = {"norm_weight": dnw, "norm_bias": dnb, "router": h.float().T @ dlogits, "w1": dw1, "w2": dw2}
        return dy + dx, grads

    def rebalance(self, plan, rate=1e-3):
        """Moves the selection bias towards experts that got fewer tokens than the mean."""
        counts = plan.counts.float()
        self.balance += rate * torch.sign(counts.mean() - counts)


def training(block, x, target, steps, rate):
    """Plain gradient descent on the squared error a token; the losses, a value each."""
    losses = []
    for _ in range(steps):
        y, saved = block.forward(x)
        diff = y.float() - target
        losses.append((diff * diff).mean())
        _, grads = block.backward((diff * (2 / len(x))).to(x.dtype), saved)
        for name, value in block.params.items():
            value.sub_((grads[name].float() * rate).to(value.dtype))
        block.rebalance(saved[7])
    return torch.stack(losses).tolist()


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, default=8192)
    ap.add_argument("--width", type=int, default=1024)
    ap.add_argument("--hidden", type=int, default=2048)
    ap.add_argument("--experts", type=int, default=32)
    ap.add_argument("--k", type=int, default=4)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--rate", type=float, default=0.1)
    a = ap.parse_args()
    block = MoEBlock(a.width, a.hidden, a.experts, a.k)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(a.tokens, a.width, device="cuda", generator=g).to(torch.bfloat16)
    target = x.float() + 0.5 * torch.randn(a.tokens, a.width, device="cuda", generator=g)
    losses = training(block, x, target, a.steps, a.rate)
    print("loss %.5f -> %.5f in %d steps" % (losses[0], losses[-1], a.steps))

    def timed(f, n=20):
        f()
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        torch.cuda.synchronize()
        start.record()
        for _ in range(n):
            f()
        end.record()
        torch.cuda.synchronize()
        return start.elapsed_time(end) / n

    def step():
        y, saved = block.forward(x)
        block.backward(y, saved)

    print("forward and backward of %d tokens: %.2f ms; forward of 4 tokens: %.3f ms" % (
        a.tokens, timed(step), timed(lambda: block.forward(x[:4]))))


if __name__ == "__main__":
    main()
