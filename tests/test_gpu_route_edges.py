"""Routing at its numeric ends: chosen experts that are masked, sigmoids that
underflow; half-precision logits.

u = 2^-24.  A weight loses |l| u of a logit l on its way into the exponential and
a few u in sums and quotients of at most n terms: (n + 2 |l| + 16) u of its value;
a gradient twice that of the sum of its terms' magnitudes.
"""

import itertools

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import mojodgl.ops as ops  # noqa: E402

U = 2.0 ** -24
INF = float("inf")
LOW = torch.finfo(torch.float32).min


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


def far_logits():
    g = torch.Generator(device="cuda").manual_seed(7)
    rows = torch.randn(40, 12, device="cuda", generator=g)
    rows[1:9] -= torch.linspace(84, 91, 8, device="cuda")[:, None]  # sigmoids around the smallest normal number
    rows[9:17] -= 250
    rows[17] = -1e4
    rows[18, ::2] = -INF
    rows[18, 1::2] -= 300
    rows[19] = -INF
    rows[20, 5] = 3.0
    rows[20, 6:] -= 200  # one expert of ordinary score among hopeless ones
    rows[21] -= torch.arange(12, device="cuda") * 20.0
    return rows


def share64(x, idx):
    """s / sum of s over the chosen, from logarithms."""
    x = np.take_along_axis(x, np.maximum(idx, 0), 1)
    x = np.where(idx < 0, -np.inf, x)
    log_s = -np.logaddexp(0, -x)
    top = np.where(np.isneginf(log_s.max(1, keepdims=True)), 0, log_s.max(1, keepdims=True))
    p = np.exp(log_s - top)
    return p / np.maximum(p.sum(1, keepdims=True), 1e-300), x


@pytest.mark.parametrize("bias", [False, True])
def test_sigmoid_weights_add_up_where_every_sigmoid_underflows(bias):
    logits = far_logits()
    k = 4
    w, i = ops.route_topk(logits, k, score="sigmoid", scale=1.5, bias=torch.zeros(12, device="cuda") if bias else None)
    idx = i.cpu().numpy()
    p, x = share64(logits.double().cpu().numpy(), idx)
    tol = (12 + 2 * np.abs(np.where(np.isfinite(x), x, 0)).max(1, keepdims=True) + 16) * U * 1.5 * p
    err = np.abs(w.double().cpu().numpy() - 1.5 * p)
    # (what is below the smallest normal number of the output's type is not held to its digits)
    assert (err <= tol + 2.0 ** -126).all(), (err - tol).max()
    assert not w[19].any() and (i[19] == -1).all()
    # the lowest finite logits are all alike
    w, i = ops.route_topk(torch.full((3, 9), LOW, device="cuda"), 4, score="sigmoid")
    assert torch.equal(w, torch.full((3, 4), 0.25, device="cuda"))


def test_sigmoid_gradients_where_every_sigmoid_underflows():
    logits = far_logits()
    grad = torch.randn(40, 4, device="cuda", generator=torch.Generator(device="cuda").manual_seed(8))
    _, i = ops.route_topk(logits, 4, score="sigmoid")
    got = ops.route_topk_backward(grad, logits, i, score="sigmoid", scale=1.5).double().cpu().numpy()
    idx, gs = i.cpu().numpy(), 1.5 * grad.double().cpu().numpy()
    p, x = share64(logits.double().cpu().numpy(), idx)
    gs = np.where(idx < 0, 0, gs)
    slope = p * np.exp(-np.logaddexp(0, np.where(np.isfinite(x), x, 0)))
    want, size = np.zeros((40, 12)), np.zeros((40, 12))
    for t in range(40):
        ok = idx[t] >= 0
        want[t, idx[t][ok]] = (slope * (gs - (p * gs).sum(1, keepdims=True)))[t][ok]
        size[t, idx[t][ok]] = (slope * (np.abs(gs) + (p * np.abs(gs)).sum(1, keepdims=True)))[t][ok]
    big = np.abs(np.where(np.isfinite(x), x, 0)).max(1, keepdims=True)
    err = np.abs(got - want)
    tol = 2 * (12 + 2 * big + 16) * U * size
    assert (err <= tol + 2.0 ** -126).all(), (err - tol).max()


@pytest.mark.parametrize("as_numpy", [False, True])
def test_float16_logits_run_in_float32(as_numpy):
    g = torch.Generator(device="cuda").manual_seed(9)
    logits, grad = torch.randn(30, 48, device="cuda", generator=g).half(), torch.randn(30, 5, device="cuda", generator=g)
    give = (lambda t: t.cpu().numpy()) if as_numpy else (lambda t: t)
    w, i = ops.route_topk(give(logits), 5)
    want_w, want_i = ops.route_topk(logits.float(), 5)
    back = ops.route_topk_backward(give(grad), give(logits), give(want_i))
    want = ops.route_topk_backward(grad, logits.float(), want_i)
    for got, ref in ((w, want_w), (i, want_i), (back, want)):
        assert torch.equal(torch.as_tensor(got).cuda(), ref)
