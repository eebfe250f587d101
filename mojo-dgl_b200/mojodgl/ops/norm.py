"""Layer norm over the last axis, forward and backward.

The reference has no dense layers; a graph transformer or mixture-of-experts
block runs its norm next to this package's grouped products, on the same
arrays.  bfloat16 tensors stay bfloat16 (statistics and sums in float32);
weight and bias may then be float32 or bfloat16.
"""

from __future__ import annotations

import math

import torch

from .. import _tensor as T
from .._lib import check, lib
from ..base import DGLError

__all__ = ["layer_norm", "layer_norm_backward"]


def _types(x, *params):
    """Element types of the rows and of the parameters."""
    present = [p for p in params if p is not None]
    if T.is_bf16(x):
        narrow = bool(present)
        for p in present:
            if not T.is_bf16(p):
                narrow = False
                if not T.is_f32(p):
                    break
        else:
            return torch.bfloat16, torch.bfloat16 if narrow else torch.float32
    dtype = T.float_type(x, *present)
    return dtype, dtype


def _stat_type(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def _check_rows(x, weight, bias):
    shape = tuple(x.shape)
    if not shape or shape[-1] < 1:
        raise DGLError("layer norm needs a last axis of at least one value, got shape {}".format(shape))
    d = shape[-1]
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and (p.ndim != 1 or p.shape[0] != d):
            raise DGLError("{} must have shape ({},), got {}".format(name, d, tuple(p.shape)))
    return shape, math.prod(shape[:-1]), d


def layer_norm(x, weight=None, bias=None, eps=1e-5, return_stats=False):
    r"""``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis.

    ``x`` is (..., D); ``weight`` and ``bias`` are (D,), a bias only together
    with a weight.  Returns an array shaped like ``x``; with ``return_stats``
    also the mean and 1 / sqrt(var + eps) of every row, which
    :func:`layer_norm_backward` takes.
    """
    if bias is not None and weight is None:
        raise DGLError("layer_norm takes a bias only together with a weight")
    if not eps >= 0:
        raise DGLError("eps must not be negative, got {}".format(eps))
    kind, (x, weight, bias) = T.operands(x, weight, bias)
    shape, rows, d = _check_rows(x, weight, bias)
    dtype, wdtype = _types(x, weight, bias)
    dev = T.device()
    xt, wt, bt = T.on(dev, x, dtype), T.on(dev, weight, wdtype), T.on(dev, bias, wdtype)
    y = torch.empty_like(xt)
    mean = rstd = None
    if return_stats:
        lead = shape[:-1]  # (sizes one by one: torch parses them faster than a tuple)
        mean = torch.empty(*lead or ((),), dtype=_stat_type(dtype), device=dev)
        rstd = torch.empty_like(mean)
    check(lib().bgl_layer_norm(T.address(xt), T.address(wt), T.address(bt), rows, d, float(eps), T.address(y),
                               T.address(mean), T.address(rstd), T.code_of(dtype), T.code_of(wdtype),
                               T.stream()), "layer_norm")
    if not return_stats:
        return T.result(y, kind)
    return T.result(y, kind), T.result(mean, kind), T.result(rstd, kind)


def layer_norm_backward(grad, x, mean, rstd, weight=None):
    r"""Gradients of :func:`layer_norm` with respect to x, weight and bias.

    ``grad`` is shaped like ``x``; ``mean`` and ``rstd`` are the forward
    call's.  Returns ``(dx, dweight, dbias)``, the last two None without a
    weight.  The sums over rows have a fixed order: the same inputs give the
    same bits.
    """
    kind, (grad, x, mean, rstd, weight) = T.operands(grad, x, mean, rstd, weight)
    shape, rows, d = _check_rows(x, weight, None)
    if T.shape_of(grad) != shape:
        raise DGLError("grad must have the shape of x, {}, got {}".format(shape, T.shape_of(grad)))
    for name, s in (("mean", mean), ("rstd", rstd)):
        if T.shape_of(s) != shape[:-1]:
            raise DGLError("{} must have shape {}, got {}".format(name, shape[:-1], T.shape_of(s)))
    if T.is_bf16(x) and T.is_bf16(grad):
        dtype, wdtype = _types(x, weight)
    else:
        present = (x, grad) if weight is None else (x, grad, weight)
        dtype = wdtype = T.float_type(*present)
    dev = T.device()
    gt, xt = T.on(dev, grad, dtype), T.on(dev, x, dtype)
    mt, rt = T.on(dev, mean, _stat_type(dtype)), T.on(dev, rstd, _stat_type(dtype))
    wt = T.on(dev, weight, wdtype)
    dx = torch.empty_like(xt)
    dw = db = ws = None
    nbytes = 0
    if weight is not None:
        dw, db = torch.empty_like(wt), torch.empty_like(wt)
        nbytes = lib().bgl_layer_norm_backward_workspace_size(rows, d, T.code_of(dtype))
        ws = T.workspace(nbytes)
    check(lib().bgl_layer_norm_backward(T.address(gt), T.address(xt), T.address(mt), T.address(rt), T.address(wt), rows,
                                        d, T.address(dx), T.address(dw), T.address(db), T.code_of(dtype),
                                        T.code_of(wdtype), T.address(ws), nbytes, T.stream()),
          "layer_norm_backward")
    if weight is None:
        return T.result(dx, kind), None, None
    return T.result(dx, kind), T.result(dw, kind), T.result(db, kind)
