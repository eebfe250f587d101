"""What a mixture-of-experts layer costs, operator by operator.

The operators are layer normalisation, the routing of tokens to experts, the sending of token rows to their experts and the
joining of what comes back, and the gradients of the experts' products.  Each case is one pass through one of them in one
direction.  ``own`` chooses who computes it: elementary torch operations in 32 bits, or the kernels of ``mojodgl.ops``.
"""

import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f32": 4}
_EPS = 1e-5
_ops = None


def _mojodgl():
    global _ops
    if _ops is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "mojo-dgl_b200"))
        from mojodgl import ops

        _ops = ops
    return _ops


# ------------------------------------------------------------------- cases
def _norm(direction, rows, width, dtype):
    return {"op": "norm", "direction": direction, "rows": rows, "width": width, "dtype": dtype}


def _route(direction, tokens, experts, k, dtype, score, bias, groups, topk_groups, group_top, renormalize, scale, masked):
    return {"op": "route", "direction": direction, "tokens": tokens, "experts": experts, "k": k, "dtype": dtype, "score": score,
            "bias": bias, "groups": groups, "topk_groups": topk_groups, "group_top": group_top, "renormalize": renormalize,
            "scale": scale, "masked": masked}


def _rows(op, tokens, experts, k, width, dtype, weighted, padded):
    return {"op": op, "tokens": tokens, "experts": experts, "k": k, "width": width, "dtype": dtype, "weighted": weighted,
            "padded": padded}


def _experts(rows, experts, d1, d2, empty):
    return {"op": "experts_backward", "rows": rows, "experts": experts, "d1": d1, "d2": d2, "dtype": "bf16", "empty": empty}


def listed():
    return [
        # the norm before the router while one sequence generates: a launch, and little else
        dict(_norm("forward", 1, 2048, "bf16"), name="norm_one_token"),
        # a full-precision evaluation batch of a width and a row count that no tile divides
        dict(_norm("forward", 20011, 1000, "f32"), name="norm_odd_f32"),
        # a training batch on its way back, with the sums over all rows for the weight and the bias
        dict(_norm("backward", 16384, 4096, "bf16"), name="norm_train_backward"),
        # a serving batch of a few sequences that each generate one token
        dict(_route("forward", 5, 64, 6, "bf16", "softmax", False, 1, 1, 1, True, 1.0, False), name="route_serve"),
        # a training batch with many small experts: sigmoid scores, a bias for balance, half of eight groups, padding tokens
        dict(_route("forward", 65536, 256, 8, "f32", "sigmoid", True, 8, 4, 2, True, 2.5, True), name="route_train_groups"),
        # the router's gradient in a training step, softmax over all experts
        dict(_route("backward", 32768, 128, 4, "f32", "softmax", False, 1, 1, 1, False, 1.0, False), name="route_train_backward"),
        # a prompt's tokens sorted by expert, and their rows sent there
        dict(_rows("dispatch", 16384, 64, 4, 2048, "bf16", False, False), name="dispatch_prompt"),
        # the experts' answers for a few generated tokens joined by the router's weights
        dict(_rows("combine", 3, 64, 8, 1024, "bf16", True, False), name="combine_serve"),
        # the same in a training step, on its way back, with padding tokens that no expert saw
        dict(_rows("combine_backward", 8191, 16, 2, 2056, "bf16", True, True), name="combine_train_backward"),
        # a fine-tuning step on one short text
        dict(_experts(190, 8, 256, 512, 1), name="experts_backward_short"),
        # relational blocks: many rows, narrow matrices, bound by memory
        dict(_experts(500000, 64, 256, 256, 2), name="experts_backward_narrow"),
        # a training batch through wide experts, bound by the tensor cores
        dict(_experts(32768, 16, 2048, 1024, 0), name="experts_backward_wide"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "route", "route", "dispatch", "combine", "combine_backward", "experts_backward", "experts_backward"])
    dtype = rng.choice(["bf16", "f32"])
    if op == "norm":
        width = _spread(rng, 33, 8192)
        return _norm(rng.choice(["forward", "backward"]), _spread(rng, 1, min(65536, (1 << 25) // width)), width, dtype)
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * _spread(rng, 4, 384 // groups)
        topk_groups = groups if groups == 1 else rng.randint(1, groups)
        k = rng.randint(1, min(10, topk_groups * (experts // groups)))
        score = rng.choice(["softmax", "sigmoid"])
        bias = score == "sigmoid" and rng.random() < 0.6
        return _route(rng.choice(["forward", "backward"]), _spread(rng, 1, 65536), experts, k, dtype, score, bias, groups, topk_groups,
                      2 if bias and groups > 1 else 1, rng.random() < 0.6, rng.choice([1.0, 2.5]), rng.random() < 0.5)
    if op == "experts_backward":
        d1, d2 = 8 * _spread(rng, 4, 192), 8 * _spread(rng, 4, 192)
        experts = _spread(rng, 1, min(96, 6 * 10 ** 7 // (d1 * d2)))
        rows = _spread(rng, 1, min(400000, 16 * 10 ** 9 // (d1 * d2), 3 * 10 ** 8 // (2 * d1 + d2)))
        return _experts(rows, experts, d1, d2, rng.randint(0, experts // 4))
    experts = _spread(rng, 4, 256)
    k, width = rng.randint(1, min(8, experts)), _spread(rng, 17, 4096)
    return _rows(op, _spread(rng, 1, min(32768, (3 << 24) // (k * width))), experts, k, width, dtype, op != "dispatch" and rng.random() < 0.7,
                 rng.random() < 0.5)


# ------------------------------------------------------------------ inputs
def _skewed_choice(tokens, experts, k, padded, g):
    """k different experts a token, some experts liked more than others; -1 throughout for padding tokens."""
    liked = torch.randn(experts, device="cuda", generator=g) * 0.7
    score = liked + torch.randn(tokens, experts, device="cuda", generator=g)
    idx = score.topk(k, dim=1).indices
    if padded:
        idx[torch.rand(tokens, device="cuda", generator=g) < 0.06] = -1
    return idx


def _lengths(rows, experts, empty, g):
    """Rows of each expert: uneven, some experts without any, all of them adding up to rows."""
    share = torch.rand(experts, generator=g) + 0.25
    share[torch.randperm(experts, generator=g)[:empty]] = 0
    ends = (share.cumsum(0) / share.sum() * rows).round().to(torch.int64)
    ends[-1] = rows
    return torch.diff(ends, prepend=torch.zeros(1, dtype=torch.int64)).clamp_(min=0)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def randn(*shape, scale=1.0, to=dtype):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(to)

    op, st = case["op"], dict(case)
    if op == "norm":
        n, d = case["rows"], case["width"]
        st["x"] = (torch.randn(n, d, device="cuda", generator=g) * (0.5 + torch.rand(n, 1, device="cuda", generator=g)) + 0.3).to(dtype)
        st["weight"] = 1 + randn(d, scale=0.1, to=torch.float32)
        st["bias"] = randn(d, scale=0.1, to=torch.float32)
        if case["direction"] == "backward":
            x = st["x"].double()
            mean = x.mean(1)
            st["mean"] = mean.float()
            st["rstd"] = (1 / ((x - mean[:, None]).square().mean(1) + _EPS).sqrt()).float()
            st["grad"] = randn(n, d, scale=0.02)
    elif op == "route":
        t, e, k = case["tokens"], case["experts"], case["k"]
        logits = randn(t, e, scale=1.5, to=torch.float32) + randn(e, scale=0.5, to=torch.float32)
        if case["masked"]:
            if e > 4 * case["groups"]:
                logits[:, e // 2] = -math.inf  # an expert that is switched off
            logits[torch.rand(t, device="cuda", generator=g) < 0.06] = -math.inf  # padding tokens
        st["logits"] = logits.to(dtype)
        st["balance"] = randn(e, scale=0.1, to=torch.float32) if case["bias"] else None
        if case["direction"] == "backward":
            x = st["logits"].float()
            best = x.sort(dim=1, descending=True, stable=True)
            st["indices"] = torch.where(best.values[:, :k] == -math.inf, -1, best.indices[:, :k])
            st["grad"] = randn(t, k, to=torch.float32)
    elif op == "experts_backward":
        n, e, d1, d2 = (case[x] for x in ("rows", "experts", "d1", "d2"))
        host = _lengths(n, e, case["empty"], torch.Generator().manual_seed(seed))
        st["seglen"], st["longest"] = host.cuda(), int(host.max())
        st["a"], st["grad"] = randn(n, d1), randn(n, d2, scale=0.1)
        st["b"] = randn(e, d1, d2, scale=1 / math.sqrt(d1))
    else:
        t, k, d = case["tokens"], case["k"], case["width"]
        st["indices"] = _skewed_choice(t, case["experts"], k, case["padded"], g)
        if op == "dispatch":
            st["x"] = randn(t, d)
        else:
            st["rows"] = randn(t * k, d)
            st["weights"] = torch.rand(t, k, device="cuda", generator=g) if case["weighted"] else None
            if op == "combine_backward":
                st["grad"] = randn(t, d, scale=0.1)
            # the places that the rows were sent to, as the layer keeps them
            st["positions"] = _plain_plan(st["indices"], case["experts"])[1]
    return st


# -------------------------------------------------------------- plain forms
def _plain_norm(st):
    x = st["x"].float()
    if st["direction"] == "forward":
        mean = x.mean(1)
        c = x - mean[:, None]
        rstd = torch.rsqrt((c * c).mean(1) + _EPS)
        y = c * rstd[:, None] * st["weight"] + st["bias"]
        return {"y": y.to(st["x"].dtype), "mean": mean, "rstd": rstd}
    grad = st["grad"].float()
    xhat = (x - st["mean"][:, None]) * st["rstd"][:, None]
    gw = grad * st["weight"]
    dx = (gw - gw.mean(1, keepdim=True) - xhat * (gw * xhat).mean(1, keepdim=True)) * st["rstd"][:, None]
    return {"dx": dx.to(st["x"].dtype), "dweight": (grad * xhat).sum(0), "dbias": grad.sum(0)}


def _plain_softmax(x):
    """Over the last axis; a row of nothing but -inf gives zeros."""
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total)


def _plain_route(st):
    x, k, groups = st["logits"].float(), st["k"], st["groups"]
    t, e = x.shape
    sigmoid = 1 / (1 + torch.exp(-x))
    c = x if st["balance"] is None else sigmoid + st["balance"]
    c = torch.where(x == -math.inf, -math.inf, c)
    if groups > 1:
        best = c.view(t, groups, e // groups).sort(dim=2, descending=True).values[:, :, : st["group_top"]]
        of_group = torch.where(best[:, :, 0] == -math.inf, -math.inf, torch.where(best == -math.inf, 0.0, best).sum(2))
        chosen = of_group.sort(dim=1, descending=True, stable=True).indices[:, : st["topk_groups"]]
        kept = torch.zeros(t, groups, dtype=torch.bool, device=x.device).scatter_(1, chosen, True)
        c = torch.where(kept[:, :, None].expand(t, groups, e // groups).reshape(t, e), c, -math.inf)
    order = c.sort(dim=1, descending=True, stable=True)
    indices = order.indices[:, :k]
    none = order.values[:, :k] == -math.inf
    if st["score"] == "softmax":
        w = _plain_softmax(torch.where(none, -math.inf, x.gather(1, indices))) if st["renormalize"] else _plain_softmax(x).gather(1, indices)
    else:
        w = torch.where(none, 0.0, sigmoid.gather(1, indices))
        if st["renormalize"]:
            w = w / w.sum(1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    return {"weights": torch.where(none, 0.0, w * st["scale"]), "indices": torch.where(none, -1, indices)}


def _plain_route_backward(st):
    x, idx = st["logits"].float(), st["indices"]
    none = idx < 0
    at = idx.clamp(min=0)
    g = torch.where(none, 0.0, st["grad"] * st["scale"])
    if st["score"] == "softmax":
        if st["renormalize"]:
            p = _plain_softmax(torch.where(none, -math.inf, x.gather(1, at)))
            dx = torch.zeros_like(x).scatter_add_(1, at, p * (g - (p * g).sum(1, keepdim=True)))
        else:
            p = _plain_softmax(x)
            dx = torch.zeros_like(x).scatter_add_(1, at, g)
            dx = p * (dx - (p * dx).sum(1, keepdim=True))
    else:
        xs = x.gather(1, at)
        s = torch.where(none, 0.0, 1 / (1 + torch.exp(-xs)))
        slope = s * (1 / (1 + torch.exp(xs)))
        if st["renormalize"]:
            total = s.sum(1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
            g = (g - (g * s).sum(1, keepdim=True) / total) / total
        dx = torch.zeros_like(x).scatter_add_(1, at, torch.where(none, 0.0, g * slope))
    return {"dlogits": dx.to(st["logits"].dtype)}


def _plain_plan(indices, experts):
    """Rows of each expert; the place that each (token, choice) goes to, those that go to no expert (~place) behind all others; and which
    of them comes to each place."""
    flat = indices.reshape(-1)
    key = torch.where(flat < 0, experts, flat)
    order = key.argsort(stable=True)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device).scatter_add_(0, key, torch.ones_like(key))[:experts]
    place = torch.empty_like(flat)
    place[order] = torch.arange(flat.numel(), device=flat.device)
    return counts, torch.where(flat < 0, ~place, place).to(torch.int32).view(indices.shape), order


def _plain_dispatch(st):
    counts, positions, order = _plain_plan(st["indices"], st["experts"])
    rows = st["x"][order // st["k"]]
    rows = torch.where((torch.arange(rows.shape[0], device=rows.device) < counts.sum())[:, None], rows, 0)
    return {"rows": rows, "counts": counts, "positions": positions}


def _plain_combine(st):
    rows, at = st["rows"], st["positions"].long()
    picked = rows[at.clamp(min=0)].float()
    w = (at >= 0).float() if st["weights"] is None else torch.where(at >= 0, st["weights"], 0.0)
    return {"y": (picked * w[:, :, None]).sum(1).to(rows.dtype)}


def _plain_combine_backward(st):
    rows, at, grad = st["rows"], st["positions"].long(), st["grad"].float()
    sent = at >= 0
    w = sent.float() if st["weights"] is None else torch.where(sent, st["weights"], 0.0)
    drows = torch.zeros(rows.shape[0] + 1, rows.shape[1], device=rows.device)
    drows[torch.where(sent, at, rows.shape[0])] = w[:, :, None] * grad[:, None, :]
    out = {"drows": drows[:-1].to(rows.dtype)}
    if st["weights"] is not None:
        out["dweights"] = torch.where(sent, (rows[at.clamp(min=0)].float() * grad[:, None, :]).sum(2), 0.0)
    return out


def _padded_place(seglen, rows):
    """For each row its segment, and its place within it."""
    ends = seglen.cumsum(0)
    row = torch.arange(rows, device=seglen.device)
    seg = torch.searchsorted(ends, row, right=True)
    return seg, row - (ends - seglen)[seg]


def _plain_experts_backward(st):
    a, b, grad = st["a"], st["b"].float(), st["grad"]
    seg, at = _padded_place(st["seglen"], a.shape[0])
    pad_a = torch.zeros(b.shape[0], st["longest"], a.shape[1], device=a.device)
    pad_g = torch.zeros(b.shape[0], st["longest"], grad.shape[1], device=a.device)
    pad_a[seg, at], pad_g[seg, at] = a.float(), grad.float()
    da = torch.bmm(pad_g, b.transpose(1, 2))[seg, at]
    return {"da": da.to(a.dtype), "db": torch.bmm(pad_a.transpose(1, 2), pad_g).to(a.dtype)}


# ---------------------------------------------------------- framework's form
def _own_norm(st):
    ops = _mojodgl()
    if st["direction"] == "forward":
        y, mean, rstd = ops.layer_norm(st["x"], st["weight"], st["bias"], eps=_EPS, return_stats=True)
        return {"y": y, "mean": mean, "rstd": rstd}
    dx, dw, db = ops.layer_norm_backward(st["grad"], st["x"], st["mean"], st["rstd"], st["weight"])
    return {"dx": dx, "dweight": dw, "dbias": db}


def _own_route(st):
    w, i = _mojodgl().route_topk(st["logits"], st["k"], score=st["score"], bias=st["balance"], num_groups=st["groups"],
                                 topk_groups=st["topk_groups"], group_top=st["group_top"], renormalize=st["renormalize"], scale=st["scale"])
    return {"weights": w, "indices": i}


def _own_route_backward(st):
    return {"dlogits": _mojodgl().route_topk_backward(st["grad"], st["logits"], st["indices"], score=st["score"],
                                                      renormalize=st["renormalize"], scale=st["scale"])}


def _own_dispatch(st):
    ops = _mojodgl()
    plan = ops.expert_plan(st["indices"], st["experts"])
    return {"rows": ops.dispatch(st["x"], plan.positions), "counts": plan.counts, "positions": plan.positions}


def _own_combine(st):
    return {"y": _mojodgl().combine(st["rows"], st["positions"], st["weights"])}


def _own_combine_backward(st):
    drows, dweights = _mojodgl().combine_backward(st["grad"], st["rows"], st["positions"], st["weights"])
    return {"drows": drows} if dweights is None else {"drows": drows, "dweights": dweights}


def _own_experts_backward(st):
    da, db = _mojodgl().segment_mm_backward(st["grad"], st["a"], st["b"], st["seglen"])
    return {"da": da, "db": db}


_PLAIN = {"norm": _plain_norm, "route": _plain_route, "route_backward": _plain_route_backward, "dispatch": _plain_dispatch,
          "combine": _plain_combine, "combine_backward": _plain_combine_backward, "experts_backward": _plain_experts_backward}
_OWN = {"norm": _own_norm, "route": _own_route, "route_backward": _own_route_backward, "dispatch": _own_dispatch,
        "combine": _own_combine, "combine_backward": _own_combine_backward, "experts_backward": _own_experts_backward}


def run(state):
    op = state["op"]
    if op == "route" and state["direction"] == "backward":
        op = "route_backward"
    return (_OWN if own else _PLAIN)[op](state)


# ------------------------------------------------------------------- floors
def work(case):
    op, size = case["op"], _BYTES[case["dtype"]]
    if op == "norm":
        n, d = case["rows"], case["width"]
        if case["direction"] == "forward":
            return {"bytes": 2 * n * d * size + 8 * d + 8 * n, "flops": 8 * n * d}
        return {"bytes": 3 * n * d * size + 12 * d + 8 * n, "flops": 14 * n * d}
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["k"]
        if case["direction"] == "forward":
            return {"bytes": t * e * size + 4 * e * case["bias"] + 12 * t * k, "flops": 4 * t * e}
        # with renormalised or sigmoid weights only the chosen experts' logits are read
        read = t * e * size if case["score"] == "softmax" and not case["renormalize"] else t * k * size
        return {"bytes": read + t * e * size + 12 * t * k, "flops": 4 * t * e}
    if op == "experts_backward":
        n, e, d1, d2 = (case[x] for x in ("rows", "experts", "d1", "d2"))
        return {"bytes": size * (2 * n * d1 + n * d2 + 2 * e * d1 * d2) + 8 * e, "flops": 4 * n * d1 * d2}
    t, k, d = case["tokens"], case["k"], case["width"]
    if op == "dispatch":
        return {"bytes": size * (t * d + t * k * d) + 12 * t * k + 8 * case["experts"], "flops": 0}
    if op == "combine":
        return {"bytes": size * (t * k * d + t * d) + (8 if case["weighted"] else 4) * t * k, "flops": 2 * t * k * d}
    # without weights the gradient of a row is its token's: the rows themselves are not read
    read = t * k * d if case["weighted"] else 0
    return {"bytes": size * (t * d + read + t * k * d) + (12 if case["weighted"] else 4) * t * k, "flops": 3 * t * k * d}


# ------------------------------------------------------------- in 64 bits
def _exact_norm(st):
    x, w = st["x"].double(), st["weight"].double()
    if st["direction"] == "forward":
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = (var + _EPS) ** -0.5
        return {"y": torch.addcmul(st["bias"].double(), (x - mean[:, None]) * rstd[:, None], w), "mean": mean, "rstd": rstd}
    dy, rstd = st["grad"].double(), st["rstd"].double()[:, None]
    n = x.shape[1]
    xhat = (x - st["mean"].double()[:, None]) * rstd
    # the vector-Jacobian product, (I - 1 1' / n - xhat xhat' / n) applied to w * dy
    v = dy * w
    dx = rstd / n * (n * v - v.sum(1, keepdim=True) - xhat * torch.einsum("ij,ij->i", v, xhat)[:, None])
    return {"dx": dx, "dweight": torch.einsum("ij,ij->j", dy, xhat), "dbias": dy.sum(0)}


def _exact_weights(x, idx, st):
    """The chosen experts' weights as a function of 64-bit logits."""
    chosen = idx >= 0
    sel = x.gather(1, idx.clamp(min=0))
    if st["score"] == "softmax":
        over = torch.where(chosen, sel, -math.inf) if st["renormalize"] else x
        w = torch.exp(sel - torch.logsumexp(over, 1, keepdim=True))
    else:
        w = torch.sigmoid(sel)
        if st["renormalize"]:
            w = w / torch.where(chosen, w, 0.0).sum(1, keepdim=True)
    return torch.where(chosen, st["scale"] * w, 0.0)


def _exact_route(st):
    x = st["logits"].double()
    if st["direction"] == "backward":
        leaf = x.clone().requires_grad_()
        alive = (x > -math.inf).any(1)
        idx = st["indices"]
        w = _exact_weights(leaf[alive], idx[alive], st)
        dx, = torch.autograd.grad(w, leaf, st["grad"][alive].double())
        return {"dlogits": dx}
    c = x if st["balance"] is None else torch.where(x == -math.inf, -math.inf, torch.sigmoid(x) + st["balance"].double())
    t, e = c.shape
    if st["groups"] > 1:
        by = c.view(t, st["groups"], -1)
        top = by.topk(min(st["group_top"], by.shape[2]), dim=2).values
        total = top.clamp(min=-1e300).where(top > -math.inf, torch.zeros_like(top)).sum(2).masked_fill(top[:, :, 0] == -math.inf, -math.inf)
        least = total.topk(st["topk_groups"], dim=1).values[:, -1:]
        c = by.masked_fill((total < least)[:, :, None], -math.inf).reshape(t, e)
    best = c.topk(st["k"], dim=1)
    idx = torch.where(best.values == -math.inf, -1, best.indices)
    w = torch.zeros(t, st["k"], dtype=torch.float64, device=x.device)
    alive = (x > -math.inf).any(1)
    w[alive] = _exact_weights(x[alive], idx[alive], st)
    return {"weights": w, "indices": None}


def _exact_rows(st):
    flat = st["indices"].reshape(-1)
    t, k = st["indices"].shape
    # where (token, choice) goes: after all of the lower experts and the earlier ones of its own
    key = torch.where(flat < 0, st["experts"], flat) * flat.numel() + torch.arange(flat.numel(), device=flat.device)
    order = key.sort().indices[: int((flat >= 0).sum())]
    token, place = order // k, torch.arange(order.numel(), device=flat.device)
    if st["op"] == "dispatch":
        rows = torch.zeros(t * k, st["width"], dtype=torch.float64, device=flat.device)
        rows[place] = st["x"].double()[token]
        return {"rows": rows, "counts": None, "positions": None}
    w = torch.ones(t, k, device=flat.device) if st["weights"] is None else st["weights"]
    w = w.double().reshape(-1)[order]
    rows = st["rows"].double()
    if st["op"] == "combine":
        return {"y": torch.zeros(t, st["width"], dtype=torch.float64, device=flat.device).index_add_(0, token, rows[place] * w[:, None])}
    grad = st["grad"].double()[token]
    drows = torch.zeros_like(rows)
    drows[place] = grad * w[:, None]
    if st["weights"] is None:
        return {"drows": drows}
    dweights = torch.zeros(t * k, dtype=torch.float64, device=flat.device)
    dweights[order] = torch.einsum("ij,ij->i", grad, rows[place])
    return {"drows": drows, "dweights": dweights.view(t, k)}


def _exact_experts(st):
    a, b, g = st["a"], st["b"], st["grad"]
    da = torch.empty(a.shape, dtype=torch.float64, device=a.device)
    db = torch.empty(b.shape, dtype=torch.float64, device=a.device)
    start = 0
    for e, n in enumerate(st["seglen"].tolist()):
        rows = slice(start, start + n)
        gs = g[rows].double()
        da[rows] = gs @ b[e].double().T
        db[e] = a[rows].double().T @ gs
        start += n
    return {"da": da, "db": db}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(st)
    if case["op"] == "route":
        return _exact_route(st)
    return _exact_experts(st) if case["op"] == "experts_backward" else _exact_rows(st)
