"""Routing, the expert plan, dispatch and combine against plain 64-bit forms.

Tolerances: u = 2^-24 for what is computed in float32 (2^-53 for float64).  A
score takes an exponential (2 u), a sum of n terms (n u) and a few roundings;
a logit l loses |l| u on its way into the exponential, so weights are held to
(n + |l| + 16) u of their value.  Dot products of n terms are held to n u times
the sum of their magnitudes; results rounded to bfloat16 get 2^-8 of their value
on top.
"""

import itertools

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import mojodgl.ops as ops  # noqa: E402
from mojodgl.base import DGLError  # noqa: E402

U32 = 2.0 ** -24
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float64: 2.0 ** -53}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float64).to(dtype)


# ------------------------------------------------------------------- routing
def scores64(x, score):
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        if score == "sigmoid":
            return 1 / (1 + np.exp(-x))
        top = x.max(1, keepdims=True)
        p = np.exp(x - np.where(np.isneginf(top), 0, top))
        total = p.sum(1, keepdims=True)
        return p / np.where(total == 0, 1, total)


def route_reference(x, k, score, bias, groups, topk_groups, group_top, renormalize, scale):
    """weights (rounded to float32, the type they come in: tiny ones underflow),
    indices, the smallest gap between what was chosen and the next best of
    every token (a decision closer than that may go either way), and c."""
    x = np.asarray(x, dtype=np.float64)
    t, e = x.shape
    s = scores64(x, score)
    by_logit = bias is None and (groups == 1 or group_top == 1)
    c = x.copy() if by_logit else s + (0 if bias is None else np.asarray(bias, dtype=np.float64))
    c[np.isneginf(x)] = -np.inf
    weights, indices, gap = np.zeros((t, k)), np.full((t, k), -1), np.full(t, np.inf)

    def closest(v, n):
        """The gap between the n best of v and their successors."""
        v = np.sort(v[~np.isneginf(v)])[::-1][: n + 1]
        return np.min(-np.diff(v)) if len(v) > 1 else np.inf

    for i in range(t):
        ci = c[i].copy()
        if groups > 1:
            by = ci.reshape(groups, -1)
            total = np.full(groups, -np.inf)
            for q in range(groups):
                best = np.sort(by[q][~np.isneginf(by[q])])[::-1][:group_top]
                if len(best):
                    total[q] = best.sum()
            gap[i] = min(gap[i], closest(total, topk_groups))
            kept = np.argsort(-total, kind="stable")[:topk_groups]
            drop = np.setdiff1d(np.arange(groups), kept)
            by[drop] = -np.inf
        order = np.argsort(-ci, kind="stable")[:k]
        order = order[~np.isneginf(ci[order])]
        gap[i] = min(gap[i], closest(ci, k))
        n = len(order)
        indices[i, :n] = order
        if not n:
            continue
        w = s[i, order]
        if renormalize:
            w = scores64(x[i, order][None], "softmax")[0] if score == "softmax" else w / w.sum()
        weights[i, :n] = scale * w
    return weights.astype(np.float32).astype(np.float64), indices, gap, c


def check_route(logits, k, near=1e-5, **opt):
    opt = dict(dict(score="softmax", bias=None, num_groups=1, topk_groups=None, group_top=1, renormalize=True, scale=1.0), **opt)
    w, i = ops.route_topk(logits, k, **opt)
    assert w.dtype == torch.float32 and i.dtype == torch.int64 and w.shape == i.shape == (logits.shape[0], k)
    bias = None if opt["bias"] is None else opt["bias"].double().cpu().numpy()
    x = logits.double().cpu().numpy()
    groups = opt["num_groups"]
    rw, ri, gap, c = route_reference(x, k, opt["score"], bias, groups, opt["topk_groups"] or groups, opt["group_top"],
                                  opt["renormalize"], opt["scale"])
    sure = (gap > near) | (gap == 0) if near else np.ones(len(gap), bool)
    got = i.cpu().numpy()
    np.testing.assert_array_equal(got[sure], ri[sure])
    if groups == 1:  # what is not sure is at least as good, place by place
        for t in np.flatnonzero(~sure):
            assert len(set(got[t])) == k and (np.abs(c[t, got[t]] - c[t, ri[t]]) <= near).all()
    finite = np.abs(np.where(np.isfinite(x), x, 0)).max(1, keepdims=True) if x.size else 0
    tol = (logits.shape[1] + 2 * finite + 16) * U32 * np.abs(rw)
    err = np.abs(w.double().cpu().numpy() - rw)
    assert (err[sure] <= tol[sure]).all(), (err[sure] - tol[sure]).max()
    return w, i


@pytest.mark.parametrize("score,renormalize", list(itertools.product(["softmax", "sigmoid"], [True, False])))
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (2, 31, 31), (9, 32, 8), (4, 33, 32), (130, 64, 6),
                                              (17, 100, 10), (65, 128, 4), (33, 256, 8), (7, 257, 8), (5, 513, 9), (3, 1024, 32)])
def test_route_sizes(score, renormalize, tokens, experts, k):
    g = gen(tokens * 1009 + experts + k)
    for dtype in (torch.float32, torch.bfloat16):
        logits = (randn(g, tokens, experts) * 2).to(dtype)
        check_route(logits, k, near=0, score=score, renormalize=renormalize, scale=1.5)  # by the logits: exact, ties included
        bias = randn(g, experts) * 0.2
        # no ties left to chance: tokens with a decision closer than float32 can see are left out
        check_route(randn(g, tokens, experts) * 2, k, score=score, renormalize=renormalize, bias=bias)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,topk_groups,group_top,k", [(8, 2, 1, 1, 2), (64, 8, 3, 2, 6), (256, 8, 4, 2, 8), (96, 32, 5, 1, 8),
                                                                    (96, 32, 5, 2, 8), (12, 12, 4, 2, 4), (20, 4, 4, 2, 7), (768, 6, 2, 1, 10),
                                                                    (1024, 32, 32, 2, 32), (18, 2, 1, 1, 9)])
def test_route_groups(score, experts, groups, topk_groups, group_top, k):
    g = gen(experts + groups)
    for bias in (None, randn(g, experts) * 0.1):
        logits = randn(g, 70, experts) * 2
        logits[5] = -float("inf")
        logits[:, experts // 3] = -float("inf")
        # softmax scores of many experts are small: their gaps too
        near = 1e-5 if score == "sigmoid" or group_top == 1 and bias is None else 2e-7
        check_route(logits, k, near=near, score=score, bias=bias, num_groups=groups, topk_groups=topk_groups, group_top=group_top)


def test_route_ties_go_to_the_lowest_index():
    g = gen(3)
    for experts, k in ((8, 3), (64, 10), (300, 12)):
        logits = torch.randint(-2, 3, (200, experts), device="cuda", generator=g).float()
        for score in ("softmax", "sigmoid"):
            check_route(logits, k, near=0, score=score)
            check_route(logits.bfloat16(), k, near=0, score=score)
        # equal logits with equal biases tie, all others are 0.01 apart and more
        bias = torch.randint(0, 2, (experts,), device="cuda", generator=g) * 0.5
        check_route(logits, k, near=0, score="sigmoid", bias=bias)
    zero = torch.zeros(4, 40, device="cuda")
    zero[:, 1::2] = -0.0
    for _, i in (check_route(zero, 6, near=0), check_route(zero, 6, near=0, num_groups=4, topk_groups=2, group_top=2)):
        assert torch.equal(i, torch.arange(6, device="cuda").expand(4, 6))


def test_route_masks():
    """Masked experts are never chosen; a token without experts gets nothing."""
    inf = float("inf")
    low = torch.finfo(torch.float32).min
    logits = torch.tensor([[-inf] * 6, [-inf, 1.0, -inf, 2.0, -inf, -inf], [low] * 6, [0.0, low, -inf, low, 1.0, -inf], [-1e4] * 6,
                           [-200.0, -300.0, -inf, -400.0, -250.0, -260.0]], device="cuda")
    for score, renormalize in itertools.product(["softmax", "sigmoid"], [True, False]):
        w, i = check_route(logits, 3, near=0, score=score, renormalize=renormalize) if score == "softmax" or not renormalize else \
            ops.route_topk(logits, 3, score=score, renormalize=renormalize)
        assert i[0].tolist() == [-1, -1, -1] and w[0].tolist() == [0, 0, 0]
        assert i[1].tolist() == [3, 1, -1] and w[1, 2] == 0
        assert i[2].tolist() == [0, 1, 2] and i[3].tolist() == [4, 0, 1]
        assert torch.isfinite(w).all()
    off = torch.zeros(6, device="cuda")
    off[3] = -inf  # a bias of -inf switches an expert off
    w, i = ops.route_topk(logits, 3, score="sigmoid", bias=off)
    assert i[1].tolist() == [1, -1, -1] and not (i == 3).any()
    # groups whose experts are all masked are not kept before others
    grouped = torch.full((1, 8), -inf, device="cuda")
    grouped[0, 5] = -3.0
    assert ops.route_topk(grouped, 2, num_groups=4, topk_groups=1, group_top=2)[1].tolist() == [[5, -1]]


def test_route_not_a_number():
    nan, inf = float("nan"), float("inf")
    logits = torch.tensor([[0.0, nan, 2.0, 1.0], [0.0, 1.0, 2.0, 3.0]], device="cuda")
    for score in ("softmax", "sigmoid"):
        w, i = ops.route_topk(logits, 2, score=score)
        assert i.tolist() == [[1, 2], [3, 2]] and w[0].isnan().all() and w[1].isfinite().all()
    w, i = ops.route_topk(logits, 2, score="sigmoid", renormalize=False)
    assert i[0].tolist() == [1, 2] and w[0, 0].isnan() and w[0, 1].isfinite()
    w, i = ops.route_topk(torch.tensor([[0.0, inf, 1.0]], device="cuda"), 2, score="sigmoid")
    assert i.tolist() == [[1, 2]] and w.isfinite().all()


def gradient_reference(x, idx, g, score, renormalize, scale):
    """The vector-Jacobian product from the formulas, and the magnitude of its terms."""
    x = np.asarray(x, dtype=np.float64)
    out, size = np.zeros_like(x), np.zeros_like(x)
    for t in range(len(x)):
        ok = [(j, e) for j, e in enumerate(idx[t]) if 0 <= e < x.shape[1]]
        if not ok:
            continue
        es = np.array([e for _, e in ok])
        gs = np.array([g[t, j] for j, _ in ok]) * scale
        if score == "softmax":
            over = es if renormalize else np.arange(x.shape[1])
            p = scores64(x[t, over][None], "softmax")[0]
            full = np.zeros(len(over))
            absfull = np.zeros(len(over))
            if renormalize:
                full, absfull = gs, np.abs(gs)
            else:
                np.add.at(full, es, gs)
                np.add.at(absfull, es, np.abs(gs))
            np.add.at(out[t], over, p * (full - (p * full).sum()))  # an expert chosen twice adds up
            np.add.at(size[t], over, p * (absfull + (p * absfull).sum()))
        else:
            s, slope = scores64(x[t, es][None], "sigmoid")[0], scores64(-x[t, es][None], "sigmoid")[0]
            if renormalize:
                total = s.sum()
                size_g = (np.abs(gs) + (np.abs(gs) * s).sum() / total) / total
                gs = (gs - (gs * s).sum() / total) / total
            else:
                size_g = np.abs(gs)
            np.add.at(out[t], es, gs * s * slope)
            np.add.at(size[t], es, size_g * s * slope)
    return out, size


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score,renormalize", list(itertools.product(["softmax", "sigmoid"], [True, False])))
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (3, 2, 2), (6, 7, 3), (2, 32, 32), (70, 33, 5), (40, 128, 4), (9, 257, 8), (3, 1024, 32)])
def test_route_backward(dtype, score, renormalize, tokens, experts, k):
    g = gen(tokens + experts * 31 + k)
    logits = (randn(g, tokens, experts) * 2).to(dtype)
    if tokens > 3:
        logits[1] = -float("inf")
        logits[2, experts // 2:] = -float("inf")
    _, idx = ops.route_topk(logits, k, score=score, renormalize=renormalize)
    grad = randn(g, tokens, k)
    got = ops.route_topk_backward(grad, logits, idx, score=score, renormalize=renormalize, scale=2.5)
    assert got.dtype == dtype and got.shape == logits.shape
    x = logits.double().cpu().numpy()
    ref, size = gradient_reference(x, idx.cpu().numpy(), grad.double().cpu().numpy(), score, renormalize, 2.5)
    big = np.abs(np.where(np.isfinite(x), x, 0)).max(1, keepdims=True)
    tol = 2 * (experts + 2 * big + 16) * U32 * size + ROUND[dtype] * np.abs(ref)
    err = np.abs(got.double().cpu().numpy() - ref)
    assert (err <= tol).all(), (err - tol).max()


def test_route_backward_skips_what_is_no_expert():
    g = gen(9)
    logits, grad = randn(g, 4, 12), randn(g, 4, 3)
    idx = torch.tensor([[0, -1, 5], [-1, -1, -1], [12, 3, 1 << 40], [7, 7, -9]], device="cuda")
    grad[0, 1] = grad[1, 0] = float("nan")  # in places without an expert
    for score, renormalize in itertools.product(["softmax", "sigmoid"], [True, False]):
        got = ops.route_topk_backward(grad, logits, idx, score=score, renormalize=renormalize).double().cpu().numpy()
        ref, size = gradient_reference(logits.double().cpu().numpy(), idx.cpu().numpy(), grad.double().cpu().numpy(), score, renormalize, 1.0)
        assert (np.abs(got - ref) <= 100 * U32 * size).all()


@pytest.mark.parametrize("score,renormalize", list(itertools.product(["softmax", "sigmoid"], [True, False])))
def test_route_backward_against_differences(score, renormalize):
    """The slopes of the 64-bit weights at fixed choices."""
    g = gen(10)
    logits, grad = randn(g, 3, 9), randn(g, 3, 4)
    _, idx = ops.route_topk(logits, 4, score=score, renormalize=renormalize)
    got = ops.route_topk_backward(grad, logits, idx, score=score, renormalize=renormalize, scale=1.25).double().cpu().numpy()
    x, at, gr = logits.double().cpu().numpy(), idx.cpu().numpy(), grad.double().cpu().numpy()

    def loss(x):
        s = np.take_along_axis(scores64(x, score), at, 1)
        return (1.25 * gr * (s / s.sum(1, keepdims=True) if renormalize else s)).sum()

    step = 1e-5
    for i in np.ndindex(x.shape):
        up, down = x.copy(), x.copy()
        up[i] += step
        down[i] -= step
        # differences: step^2 of a third derivative below 100, 1e-15 / step of rounding; float32 gradients: 100 u of terms below 8
        assert abs((loss(up) - loss(down)) / (2 * step) - got[i]) < 2e-8 + 800 * U32


def test_route_strides_streams_and_numpy():
    g = gen(12)
    base = randn(g, 60, 130)
    for x in (base[:, 1:65], base[::3, :64], base.t()[:64], base[:1, :64].expand(7, 64)):
        got, want = ops.route_topk(x, 4), ops.route_topk(x.contiguous().clone(), 4)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    w, i = ops.route_topk(base.cpu().numpy(), 5)
    assert isinstance(w, np.ndarray) and i.dtype == np.int64
    np.testing.assert_array_equal(i, ops.route_topk(base, 5)[1].cpu().numpy())
    side = torch.cuda.Stream()
    late, big = torch.zeros_like(base), torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(4):
            big = big @ big * 1e-2
        late.copy_(base)
        w2, i2 = ops.route_topk(late, 5)
        plan = ops.expert_plan(i2, 130)
        rows = ops.dispatch(late, plan.positions)
    side.synchronize()
    assert torch.equal(i2, ops.route_topk(base, 5)[1])
    assert torch.equal(rows, ops.dispatch(base, ops.expert_plan(i2, 130).positions))


# ---------------------------------------------------------------------- plan
def check_plan(idx, experts):
    plan = ops.expert_plan(idx, experts)
    flat = idx.reshape(-1).cpu().numpy().astype(np.int64)
    bins = np.where((flat < 0) | (flat >= experts), experts, flat)
    order = np.argsort(bins, kind="stable")
    place = np.empty(len(flat), dtype=np.int64)
    place[order] = np.arange(len(flat))
    place = np.where(bins == experts, ~place, place)
    assert plan.counts.dtype == torch.int64 and plan.positions.dtype == torch.int32
    np.testing.assert_array_equal(plan.counts.cpu().numpy(), np.bincount(bins, minlength=experts + 1)[:experts])
    np.testing.assert_array_equal(plan.positions.cpu().numpy().reshape(-1), place)
    return plan


@pytest.mark.parametrize("tokens,k", [(0, 3), (1, 1), (1, 8), (31, 1), (11, 3), (64, 1), (341, 3), (512, 2), (1025, 1), (1000, 8),
                                      (5000, 7), (70001, 3), (300000, 8)])
def test_plan_sizes(tokens, k):
    g = gen(tokens + k)
    for experts in (1, 2, 31, 64, 257, 1024, 8191) if tokens < 100000 else (3, 384, 8191):
        idx = torch.randint(-1, experts + 1, (tokens, k), device="cuda", generator=g)
        check_plan(idx, experts)
        check_plan((idx % 3).to(torch.int32), experts)  # crowded: three experts get all, or there are fewer
    check_plan(torch.full((tokens, k), -1, device="cuda"), 5)
    check_plan(torch.full((tokens, k), 1 << 40, device="cuda"), 5)


# -------------------------------------------------------- dispatch and combine
def rows_case(seed, tokens, k, d, dtype, experts=6, padded=0.2):
    g = gen(seed)
    idx = torch.randint(0, experts, (tokens, k), device="cuda", generator=g)
    idx[torch.rand(tokens, k, device="cuda", generator=g) < padded] = -1
    plan = ops.expert_plan(idx, experts)
    wtype = torch.float64 if dtype == torch.float64 else torch.float32
    return (randn(g, tokens, d, dtype=dtype), randn(g, tokens * k, d, dtype=dtype), plan.positions, randn(g, tokens, k, dtype=wtype))


SIZES = [(0, 2, 8), (1, 1, 1), (1, 8, 1024), (3, 8, 1000), (5, 2, 7), (9, 3, 33), (70, 4, 64), (33, 1, 260), (17, 6, 2056), (300, 2, 129),
         (2, 32, 96), (2, 40, 24), (5, 3, 5000), (3, 2, 20001), (4000, 2, 16)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("tokens,k,d", SIZES)
def test_rows(dtype, tokens, k, d):
    x, rows, pos, w = rows_case(tokens * 31 + d, tokens, k, d, dtype)
    p = pos.long()
    sent, at = p >= 0, torch.where(p >= 0, p, ~p)
    # dispatch: every row is written once
    want = torch.empty_like(rows)
    want[at] = torch.where(sent[:, :, None], x[:, None, :].expand(tokens, k, d), torch.zeros((), dtype=dtype, device="cuda"))
    assert torch.equal(ops.dispatch(x, pos), want)
    u = 2.0 ** (-53 if dtype == torch.float64 else -24)
    for weights in (w, None):
        if weights is not None:
            weights = torch.where(sent, weights, float("nan"))  # not read: these pairs have no expert
        spoiled = rows.clone()
        spoiled[at[~sent]] = float("nan")
        ww = torch.where(sent, w if weights is not None else 1.0, 0.0).double()
        clean = torch.where(sent[:, :, None], spoiled[at], 0).double()
        terms = clean * ww[:, :, None]
        ref = terms.sum(1)
        y = ops.combine(spoiled, pos, weights)
        assert y.dtype == dtype and y.shape == (tokens, d)
        assert ((y.double() - ref).abs() <= (k + 2) * u * terms.abs().sum(1) + ROUND[dtype] * ref.abs()).all()
        drows, dw = ops.combine_backward(x, spoiled, pos, weights)
        ref = torch.zeros(tokens * k, d, dtype=torch.float64, device="cuda")
        ref[at] = ww[:, :, None] * x.double()[:, None, :]
        assert drows.dtype == dtype
        assert ((drows.double() - ref).abs() <= (2 * u + ROUND[dtype]) * ref.abs()).all()
        if weights is None:
            assert dw is None
            continue
        terms = clean * x.double()[:, None, :]
        assert dw.dtype == w.dtype and dw.shape == (tokens, k)
        assert ((dw.double() - terms.sum(2)).abs() <= (d + 4) * u * terms.abs().sum(2)).all()
        assert torch.equal(dw, ops.combine_backward(x, spoiled, pos, weights)[1])


def test_rows_strides_and_alignment():
    g = gen(21)
    _, _, pos, w = rows_case(1, 40, 3, 8, torch.float32)
    base, tall = randn(g, 40, 300), randn(g, 120, 300)
    for cut in (slice(1, 257), slice(0, 256), slice(3, 20)):
        x, rows = base[:, cut], tall[:, cut]
        assert torch.equal(ops.dispatch(x, pos), ops.dispatch(x.clone(), pos))
        assert torch.equal(ops.combine(rows, pos, w), ops.combine(rows.clone(), pos, w))
        for p, q in zip(ops.combine_backward(x, rows, pos, w.t().contiguous().t()), ops.combine_backward(x.clone(), rows.clone(), pos, w)):
            assert torch.equal(p, q)
    flat = randn(g, 120 * 64 + 8, dtype=torch.bfloat16)
    for shift in (1, 2, 4):
        rows = flat[shift:shift + 120 * 64].view(120, 64)
        assert torch.equal(ops.combine(rows, pos, w), ops.combine(rows.clone(), pos, w))
        assert torch.equal(ops.dispatch(rows[:40], pos), ops.dispatch(rows[:40].clone(), pos))
    token = randn(g, 1, 64).expand(40, 64)
    assert torch.equal(ops.dispatch(token, pos), ops.dispatch(token.clone(), pos))
    assert isinstance(ops.combine(tall.cpu().numpy(), pos.cpu().numpy(), w.cpu().numpy()), np.ndarray)


def test_rows_against_differences():
    x, rows, pos, w = rows_case(5, 4, 3, 5, torch.float64)
    dy = x
    drows, dw = ops.combine_backward(dy, rows, pos, w)
    dx = ops.combine(rows, pos)  # the gradient of dispatch, rows standing for the gradient of what it sent
    step = 1e-6

    def slope(t, i, f):
        keep = float(t.view(-1)[i])
        t.view(-1)[i] = keep + step
        up = float(f())
        t.view(-1)[i] = keep - step
        down = float(f())
        t.view(-1)[i] = keep
        return (up - down) / (2 * step)

    for t, grad, f in ((rows, drows, lambda: (ops.combine(rows, pos, w) * dy).sum()), (w, dw, lambda: (ops.combine(rows, pos, w) * dy).sum())):
        for i in range(t.numel()):
            assert abs(slope(t, i, f) - float(grad.view(-1)[i])) < 1e-8  # linear: 1e-15 * 50 / step of rounding
    z = torch.randn_like(x)
    for i in range(z.numel()):
        assert abs(slope(z, i, lambda: (ops.dispatch(z, pos) * rows).sum()) - float(dx.view(-1)[i])) < 1e-8


def test_positions_that_no_plan_gives_are_skipped():
    x, rows, pos, w = rows_case(6, 4, 2, 16, torch.float32)
    bad = torch.tensor([[8, -9], [2 ** 31 - 1, -2 ** 31], [0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    assert not ops.combine(rows, bad, w)[:2].any()
    assert torch.equal(ops.dispatch(x, bad)[:4], x[[2, 2, 3, 3]])
    drows, dw = ops.combine_backward(x, rows, bad, w)
    assert not dw[:2].any() and torch.equal(drows[0], w[2, 0] * x[2])


def test_more_than_two_to_the_31_values():
    """Rows at the end of arrays whose offsets need 64 bits."""
    tokens, k, d = 300000, 8, 1024
    g = gen(23)
    idx = torch.randint(0, 64, (tokens, k), device="cuda", generator=g)
    pos = ops.expert_plan(idx, 64).positions
    x = randn(g, 1, d, dtype=torch.bfloat16).repeat(tokens, 1)
    x[-5:] = randn(g, 5, d, dtype=torch.bfloat16)
    rows = ops.dispatch(x, pos)
    probe = torch.cat([pos[-5:].reshape(-1).long(), torch.tensor([tokens * k - 1, tokens * k - 2], device="cuda")])
    owner = torch.empty(tokens * k, dtype=torch.int64, device="cuda")
    owner[pos.reshape(-1).long()] = torch.arange(tokens * k, device="cuda") // k
    assert torch.equal(rows[probe], x[owner[probe]])
    w = torch.rand(tokens, k, device="cuda", generator=g)
    y = ops.combine(rows, pos, w)
    want = (x[-5:].double() * w[-5:].double().sum(1, keepdim=True))
    assert ((y[-5:].double() - want).abs() <= (2.0 ** -8 + 10 * U32) * want.abs()).all()
    drows, dw = ops.combine_backward(x, rows, pos, w)
    want = w.view(-1)[torch.argsort(pos.reshape(-1))][probe][:, None].double() * x[owner[probe]].double()
    assert ((drows[probe].double() - want).abs() <= (2.0 ** -8 + 4 * U32) * want.abs()).all()
    del rows, drows, y
    tokens, experts = (1 << 22) + 3, 520
    logits = torch.zeros(tokens, experts, dtype=torch.bfloat16, device="cuda")
    logits[-3:] = randn(g, 3, experts, dtype=torch.bfloat16)
    w, i = ops.route_topk(logits, 4)
    small = ops.route_topk(logits[-3:].clone(), 4)
    assert torch.equal(w[-3:], small[0]) and torch.equal(i[-3:], small[1])
    grad = torch.ones(tokens, 4, device="cuda")
    back = ops.route_topk_backward(grad, logits, i, renormalize=False)
    assert torch.equal(back[-3:], ops.route_topk_backward(grad[-3:], logits[-3:].clone(), i[-3:], renormalize=False))


def test_refusals():
    x = torch.zeros(4, 8, device="cuda")
    pos = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    rows = torch.zeros(8, 8, device="cuda")
    w = torch.zeros(4, 2, device="cuda")
    for call in (lambda: ops.route_topk(x.double(), 2), lambda: ops.route_topk(x.long(), 2), lambda: ops.route_topk(x[0], 1),
                 lambda: ops.route_topk(x, 0), lambda: ops.route_topk(x, 9), lambda: ops.route_topk(x, 2, score="top"),
                 lambda: ops.route_topk(x, 2, num_groups=3), lambda: ops.route_topk(x, 2, num_groups=0),
                 lambda: ops.route_topk(x, 3, num_groups=4, topk_groups=1), lambda: ops.route_topk(x, 2, num_groups=2, topk_groups=3),
                 lambda: ops.route_topk(x, 2, num_groups=2, group_top=3), lambda: ops.route_topk(x, 2, bias=torch.zeros(7, device="cuda")),
                 lambda: ops.route_topk(torch.zeros(2, 1025, device="cuda"), 2), lambda: ops.route_topk(torch.zeros(2, 100, device="cuda"), 33),
                 lambda: ops.route_topk(torch.zeros(2, 99, device="cuda"), 3, num_groups=33),
                 lambda: ops.route_topk_backward(w, x, pos[:3]), lambda: ops.route_topk_backward(w[:, :1], x, pos),
                 lambda: ops.route_topk_backward(w, x, pos, score="max"),
                 lambda: ops.expert_plan(pos[0], 4), lambda: ops.expert_plan(pos, 0), lambda: ops.expert_plan(pos, 8192),
                 lambda: ops.expert_plan(pos + 0.5, 4),
                 lambda: ops.dispatch(x[:3], pos), lambda: ops.dispatch(x, pos.float()), lambda: ops.dispatch(x[0], pos),
                 lambda: ops.combine(rows[:7], pos), lambda: ops.combine(rows, pos, w[:, :1]), lambda: ops.combine(rows, pos[0]),
                 lambda: ops.combine_backward(x[:, :4], rows, pos, w), lambda: ops.combine_backward(x, rows, pos, w[:2])):
        with pytest.raises(DGLError):
            call()
