"""The operators of a mixture-of-experts layer together, as examples/moe_block.py
runs them: against automatic differentiation of the same block in float64, and a
few steps of training."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("moe_block", os.path.join(ROOT, "examples", "moe_block.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def reference(block, x, dy, indices, active, answers):
    """The block in float64 with the given choice of experts and the given
    active hidden units (both are decided in bfloat16, where a unit within a
    rounding of zero may fall on either side), and its gradients.  The experts'
    answers have the values that the block kept, in bfloat16: the router's
    gradient is a difference of their products with dy, in which a rounding of
    theirs can be all that is left for a single token."""
    p = {k: v.double().requires_grad_() for k, v in block.params.items()}
    leaf = x.double().requires_grad_()
    h = torch.nn.functional.layer_norm(leaf, leaf.shape[1:], p["norm_weight"], p["norm_bias"])
    s = torch.sigmoid(h @ p["router"]).gather(1, indices)
    w = s / s.sum(1, keepdim=True)
    rows = torch.einsum("td,tkdh->tkh", h, p["w1"][indices]) * active
    out = torch.einsum("tkh,tkhd->tkd", rows, p["w2"][indices])
    assert (out - answers).norm() <= 2.0 ** -5 * out.norm()
    y = leaf + ((out + (answers - out).detach()) * w[:, :, None]).sum(1)
    grads = torch.autograd.grad(y, [leaf, *p.values()], dy.double())
    return y.detach(), grads[0], dict(zip(p, grads[1:]))


@pytest.mark.parametrize("tokens,width,hidden,experts,k", [(1, 64, 96, 4, 2), (37, 72, 40, 5, 3), (300, 128, 256, 16, 4)])
def test_block_against_float64(example, tokens, width, hidden, experts, k):
    block = example.MoEBlock(width, hidden, experts, k, seed=tokens)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    block.balance += torch.randn(experts, device="cuda", generator=g) * 0.05
    block.params["norm_weight"] += torch.randn(width, device="cuda", generator=g) * 0.1
    x, dy = (torch.randn(tokens, width, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    y, saved = block.forward(x)
    dx, grads = block.backward(dy, saved)
    at, a1, a2 = saved[7].positions.long(), saved[9], saved[10]
    ry, rdx, rgrads = reference(block, x, dy, saved[6], (a1 > 0)[at], a2[at].double())

    def near(got, want):
        # bf16 activations: up to ten roundings of 2^-9 on the way, 2^-5 of the norm leaves room for all of them
        return (got.double() - want).norm() <= 2.0 ** -5 * want.norm()

    assert near(y, ry) and near(dx, rdx)
    for name, want in rgrads.items():
        assert grads[name].shape == want.shape and near(grads[name], want), name


def test_training_lowers_the_loss(example):
    block = example.MoEBlock(128, 256, 8, 2)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(512, 128, device="cuda", generator=g).to(torch.bfloat16)
    target = x.float() + 0.5 * torch.randn(512, 128, device="cuda", generator=g)
    losses = example.training(block, x, target, steps=12, rate=0.1)
    assert losses[-1] < 0.97 * losses[0]
    assert torch.isfinite(torch.tensor(losses)).all()
