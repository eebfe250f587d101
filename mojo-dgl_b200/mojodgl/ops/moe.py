"""Routing of tokens to experts, and the rows that go there and come back.

A mixture-of-experts layer on this package's grouped products::

    weights, indices = route_topk(x @ router, k)
    plan = expert_plan(indices, num_experts)
    rows = dispatch(x, plan.positions)                 # sorted by expert
    rows = segment_mm(rows, expert_weights, plan.counts)
    y = combine(rows, plan.positions, weights)

``segment_mm_backward``, ``combine_backward`` and ``route_topk_backward`` lead
back; the gradient of ``dispatch`` is ``combine`` without weights.  None of the
functions here waits for the device (indices given as floats excepted, which are
checked to be whole numbers), nor does ``segment_mm_backward``; ``segment_mm`` reads
``counts`` back to check them.
"""

from __future__ import annotations

from typing import NamedTuple

import numpy as np
import torch

from .. import _tensor as T
from .._lib import SCORES, check, lib
from ..base import DGLError

__all__ = ["route_topk", "route_topk_backward", "ExpertPlan", "expert_plan", "dispatch", "combine",
           "combine_backward"]


# -------------------------------------------------------------------- routing
def _logits(logits):
    """The logits as float32 or bfloat16, with their element type."""
    if logits.ndim != 2:
        raise DGLError("logits must be (tokens, experts), got shape {}".format(T.shape_of(logits)))
    if T.is_bf16(logits):
        return torch.bfloat16
    if T.is_f32(logits) or str(logits.dtype).endswith("float16"):
        return torch.float32
    raise DGLError("logits must be float32, bfloat16 or float16, got {}".format(logits.dtype))


def _score(score):
    if score not in SCORES:
        raise DGLError("score must be 'softmax' or 'sigmoid', got {!r}".format(score))
    return SCORES[score]


def _choices(k, experts):
    k = int(k)
    if not 1 <= k <= experts:
        raise DGLError("k must be in [1, {}], got {}".format(experts, k))
    return k


def route_topk(logits, k, *, score="softmax", bias=None, num_groups=1, topk_groups=None,
               group_top=1, renormalize=True, scale=1.0):
    r"""The ``k`` best experts of every token and the weights of their answers.

    ``logits`` is (tokens, experts).  An expert's score s is the softmax of the
    token's logits or their sigmoid; c = s + ``bias`` (a (experts,) array, for
    balance) decides which experts are chosen, s what they weigh.  With
    ``num_groups`` the experts form equal runs; a run counts the sum of its
    ``group_top`` (1 or 2) best c, and only experts of the ``topk_groups`` best
    runs (default: all) are chosen.  Ties go to the lower index.  The weights
    are ``scale`` * s, divided by their sum first if ``renormalize``.

    A logit of -inf masks its expert.  A token with fewer than ``k`` experts
    left (a padding token has none) gets index -1 and weight 0 in the remaining
    places.  Returns (weights, indices), float32 and int64, both (tokens, k).
    """
    kind, (logits, bias) = T.operands(logits, bias)
    dtype = _logits(logits)
    tokens, experts = logits.shape
    k, code = _choices(k, experts), _score(score)
    num_groups = int(num_groups)
    topk_groups = num_groups if topk_groups is None else int(topk_groups)
    if num_groups < 1 or experts % num_groups:
        raise DGLError("num_groups must divide the {} experts, got {}".format(experts, num_groups))
    if not 1 <= topk_groups <= num_groups:
        raise DGLError("topk_groups must be in [1, {}], got {}".format(num_groups, topk_groups))
    if group_top not in (1, 2):
        raise DGLError("group_top must be 1 or 2, got {}".format(group_top))
    if k > topk_groups * (experts // num_groups):
        raise DGLError("k is {}, but the kept groups have {} experts".format(
            k, topk_groups * (experts // num_groups)))
    if bias is not None and T.shape_of(bias) != (experts,):
        raise DGLError("bias must have shape ({},), got {}".format(experts, T.shape_of(bias)))
    dev = T.device()
    lt, bt = T.on(dev, logits, dtype), T.on(dev, bias, torch.float32)
    weights = torch.empty(tokens, k, dtype=torch.float32, device=dev)
    indices = torch.empty_like(weights, dtype=torch.int64)
    check(lib().bgl_route_topk(T.address(lt), T.address(bt), tokens, experts, k, code, num_groups,
                               topk_groups, group_top, int(bool(renormalize)), float(scale),
                               T.address(weights), T.address(indices), T.code_of(dtype), T.stream()),
          "route_topk")
    return T.result(weights, kind), T.result(indices, kind)


def route_topk_backward(grad, logits, indices, *, score="softmax", renormalize=True, scale=1.0):
    r"""Gradient of :func:`route_topk`'s weights with respect to the logits.

    ``grad`` is the gradient of the weights, (tokens, k), ``indices`` the
    chosen experts; the other arguments are the forward call's.  The choice
    itself, and so the bias, has no gradient.  Places with index -1 (any index
    that is not an expert's) have none either, nor have masked experts (logits of
    -inf) that a choice made elsewhere holds.  Returns (tokens, experts) in the
    logits' type, float32 for float16 logits.
    """
    kind, (grad, logits, indices) = T.operands(grad, logits, indices)
    dtype = _logits(logits)
    tokens, experts = logits.shape
    shape = T.shape_of(indices)
    if len(shape) != 2 or shape[0] != tokens:
        raise DGLError("indices must be ({}, k), got shape {}".format(tokens, shape))
    k, code = _choices(shape[1], experts), _score(score)
    if T.shape_of(grad) != shape:
        raise DGLError("grad must have the shape of indices, {}, got {}".format(shape, T.shape_of(grad)))
    indices = T.ids(indices)
    dev = T.device()
    gt, lt = T.on(dev, grad, torch.float32), T.on(dev, logits, dtype)
    it = T.on(dev, indices, torch.int64)
    dlogits = torch.empty_like(lt)
    check(lib().bgl_route_topk_backward(T.address(gt), T.address(lt), T.address(it), tokens, experts, k, code,
                                        int(bool(renormalize)), float(scale), T.address(dlogits),
                                        T.code_of(dtype), T.stream()), "route_topk_backward")
    return T.result(dlogits, kind)


# ------------------------------------------------------------ rows and experts
class ExpertPlan(NamedTuple):
    """Where :func:`dispatch` sends rows: ``counts[e]`` rows to expert e (int64,
    what ``segment_mm`` takes as ``seglen_a``), choice j of token t to row
    ``positions[t, j]`` (int32).  A choice without an expert has a row behind
    all others, stored as ``~row``."""

    counts: object
    positions: object


def expert_plan(indices, num_experts):
    r"""Sorts the choices by expert, the earlier one first among equals.

    ``indices`` is (tokens, k); an index outside [0, ``num_experts``), such as
    the -1 of a padding token, goes to no expert.
    """
    kind, (indices,) = T.operands(indices)
    if len(T.shape_of(indices)) != 2:
        raise DGLError("indices must be (tokens, k), got shape {}".format(T.shape_of(indices)))
    experts = int(num_experts)
    if experts < 1:
        raise DGLError("num_experts must be positive, got {}".format(experts))
    indices = T.ids(indices)
    dev = T.device()
    it = T.on(dev, indices, torch.int64)
    items = it.numel()
    counts = torch.empty(experts, dtype=torch.int64, device=dev)
    positions = torch.empty_like(it, dtype=torch.int32)
    nbytes = lib().bgl_expert_plan_workspace_size(items, experts)
    ws = T.workspace(nbytes) if nbytes else None
    check(lib().bgl_expert_plan(T.address(it), items, experts, T.address(counts), T.address(positions),
                                T.address(ws), nbytes, T.stream()), "expert_plan")
    return ExpertPlan(T.result(counts, kind), T.result(positions, kind))


def _positions(positions):
    shape = positions.shape
    if len(shape) != 2:
        raise DGLError("positions must be (tokens, k), got shape {}".format(tuple(shape)))
    if positions.dtype is torch.int32:
        return shape
    if T.is_torch(positions):
        whole = not (positions.is_floating_point() or positions.is_complex()
                     or positions.dtype == torch.bool)
    else:
        whole = np.issubdtype(positions.dtype, np.integer)
    if not whole:
        raise DGLError("positions must be whole numbers, got {}".format(positions.dtype))
    return shape


def _places(dev, positions):
    """The positions as int32 on the device; those beyond its range at its ends,
    which lie outside all rows (a cast alone would take their low halves)."""
    if positions.dtype is torch.int32:
        return T.on(dev, positions, torch.int32)
    low, high = -2 ** 31, 2 ** 31 - 1
    if T.is_torch(positions):
        positions = positions.to(torch.int64).clamp(low, high)
    elif positions.dtype != np.int32:
        span = np.iinfo(positions.dtype)
        positions = positions.clip(max(low, span.min), min(high, span.max)).astype(np.int32)
    return T.on(dev, positions, torch.int32)


def _matrix(x, what, rows):
    shape = x.shape
    if len(shape) != 2 or shape[0] != rows:
        raise DGLError("{} must be ({}, D), got shape {}".format(what, rows, tuple(shape)))
    return shape[1]


def _weights(weights, tokens, k):
    if weights is not None and tuple(weights.shape) != (tokens, k):
        raise DGLError("weights must be ({}, {}), got shape {}".format(tokens, k, T.shape_of(weights)))


def _weight_type(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def dispatch(x, positions):
    r"""Sends every token's row to its places: ``rows[positions[t, j]] = x[t]``.

    ``x`` is (tokens, D).  Returns (tokens * k, D), sorted by expert; the rows
    of choices without an expert, behind all others, are zeros.  The gradient
    with respect to x is ``combine(grad, positions)``.
    """
    kind, (x, positions) = T.operands(x, positions)
    tokens, k = _positions(positions)
    d = _matrix(x, "x", tokens)
    dtype = T.float_type(x)
    dev = T.device()
    xt, pt = T.on(dev, x, dtype), _places(dev, positions)
    rows = xt.new_empty(tokens * k, d)
    check(lib().bgl_dispatch_rows(T.address(xt), T.address(pt), tokens, k, d, T.address(rows),
                                  T.code_of(dtype), T.stream()), "dispatch")
    return T.result(rows, kind)


def combine(rows, positions, weights=None):
    r"""Joins what the experts answered:
    ``y[t] = sum_j weights[t, j] * rows[positions[t, j]]``.

    ``rows`` is (tokens * k, D), ``weights`` (tokens, k) or None for ones;
    choices without an expert add nothing, whatever their weight.  Sums run in
    float32 (float64 for float64 rows) in the order of the choices.
    """
    kind, (rows, positions, weights) = T.operands(rows, positions, weights)
    tokens, k = _positions(positions)
    d = _matrix(rows, "rows", tokens * k)
    _weights(weights, tokens, k)
    dtype = T.float_type(rows)
    dev = T.device()
    rt, pt = T.on(dev, rows, dtype), _places(dev, positions)
    wt = T.on(dev, weights, _weight_type(dtype))
    y = rt.new_empty(tokens, d)
    check(lib().bgl_combine_rows(T.address(rt), T.address(pt), T.address(wt), tokens, k, d, T.address(y),
                                 T.code_of(dtype), T.stream()), "combine")
    return T.result(y, kind)


def combine_backward(grad, rows, positions, weights=None):
    r"""Gradients of :func:`combine` with respect to the rows and the weights:
    ``drows[positions[t, j]] = weights[t, j] * grad[t]`` and
    ``dweights[t, j] = <grad[t], rows[positions[t, j]]>``.

    Choices without an expert get rows of zeros and a weight gradient of 0.
    Returns (drows, dweights), the latter None without weights.
    """
    kind, (grad, rows, positions, weights) = T.operands(grad, rows, positions, weights)
    tokens, k = _positions(positions)
    d = _matrix(rows, "rows", tokens * k)
    if T.shape_of(grad) != (tokens, d):
        raise DGLError("grad must be ({}, {}), got shape {}".format(tokens, d, T.shape_of(grad)))
    _weights(weights, tokens, k)
    dtype = T.float_type(grad, rows)
    dev = T.device()
    gt, rt, pt = T.on(dev, grad, dtype), T.on(dev, rows, dtype), _places(dev, positions)
    wt = T.on(dev, weights, _weight_type(dtype))
    drows = torch.empty_like(rt)
    dweights = None
    if weights is not None:
        dweights = torch.empty_like(wt)
    check(lib().bgl_combine_rows_backward(T.address(gt), T.address(rt), T.address(pt), T.address(wt), tokens, k, d,
                                          T.address(drows), T.address(dweights), T.code_of(dtype),
                                          T.stream()), "combine_backward")
    return T.result(drows, kind), None if weights is None else T.result(dweights, kind)
