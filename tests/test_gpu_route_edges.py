"""Gradients of routing at experts that are masked."""

import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

import mojodgl.ops as ops  # noqa: E402

INF = float("inf")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score,renormalize", list(itertools.product(["softmax", "sigmoid"], [True, False])))
@pytest.mark.parametrize("experts,k", [(5, 3), (64, 6), (130, 4), (257, 8), (1000, 32)])
def test_chosen_experts_that_are_masked_have_no_gradient(dtype, score, renormalize, experts, k):
    """Choices made elsewhere may hold experts whose logit is -inf."""
    g = torch.Generator(device="cuda").manual_seed(experts + k)
    logits = torch.randn(6, experts, device="cuda", generator=g).to(dtype)
    idx = torch.rand(6, experts, device="cuda", generator=g).topk(k).indices
    grad = torch.randn(6, k, device="cuda", generator=g)
    clean = ops.route_topk_backward(grad, logits, idx, score=score, renormalize=renormalize)
    logits[1] = -INF  # a padding token
    logits[3].scatter_(0, idx[3], -INF)  # every chosen expert
    logits[4, idx[4, 0]] = -INF  # one of them
    got = ops.route_topk_backward(grad, logits, idx, score=score, renormalize=renormalize)
    assert not got[[1, 3]].any()  # (NaN counts as something)
    assert torch.isfinite(got).all() and got[4, idx[4, 0]] == 0
    assert torch.equal(got[[0, 2, 5]], clean[[0, 2, 5]])
