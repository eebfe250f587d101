"""Argument checks of the mixture-of-experts operators, and what happens without
a device; no kernel runs here."""

import ctypes

import numpy as np
import pytest
import torch

import mojodgl.ops as ops
from mojodgl import _lib
from mojodgl.base import DGLError

INVALID, UNSUPPORTED, WORKSPACE = 1, 3, 4


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
@pytest.mark.parametrize("as_torch", [False, True])
def test_no_cpu_fallback_without_a_device(as_torch):
    def a(*shape, dtype=np.float32):
        v = np.zeros(shape, dtype)
        return torch.from_numpy(v) if as_torch else v

    pos = a(4, 2, dtype=np.int32)
    for call in (lambda: ops.layer_norm(a(4, 8)), lambda: ops.layer_norm_backward(a(4, 8), a(4, 8), a(4), a(4), a(8)),
                 lambda: ops.route_topk(a(4, 8), 2), lambda: ops.route_topk_backward(a(4, 2), a(4, 8), pos),
                 lambda: ops.expert_plan(pos, 3), lambda: ops.dispatch(a(4, 8), pos), lambda: ops.combine(a(8, 8), pos),
                 lambda: ops.combine_backward(a(4, 8), a(8, 8), pos, a(4, 2)),
                 lambda: ops.segment_mm_backward(a(5, 3), a(5, 4), a(2, 4, 3), np.array([2, 3]))):
        with pytest.raises(DGLError, match="CUDA device"):
            call()


def test_refusals_come_before_the_device():
    x, pos = np.zeros((4, 8), np.float32), np.zeros((4, 2), np.int32)
    for call, says in ((lambda: ops.layer_norm(x, bias=np.zeros(8)), "only together"), (lambda: ops.layer_norm(x, np.zeros(7)), "weight"),
                       (lambda: ops.layer_norm(np.zeros((3, 0))), "last axis"), (lambda: ops.layer_norm(x, eps=-1), "eps"),
                       (lambda: ops.layer_norm_backward(x[:2], x, np.zeros(4), np.zeros(4)), "grad"),
                       (lambda: ops.layer_norm_backward(x, x, np.zeros(3), np.zeros(4)), "mean"),
                       (lambda: ops.route_topk(x.astype(np.float64), 2), "float32"), (lambda: ops.route_topk(x, 9), "k must"),
                       (lambda: ops.route_topk(x, 2, score="best"), "softmax"), (lambda: ops.route_topk(x, 2, num_groups=3), "num_groups"),
                       (lambda: ops.route_topk(x, 2, num_groups=4, topk_groups=5), "topk_groups"),
                       (lambda: ops.route_topk(x, 3, num_groups=4, topk_groups=1), "kept groups"),
                       (lambda: ops.route_topk(x, 2, group_top=0), "group_top"), (lambda: ops.route_topk(x, 2, bias=np.zeros(7)), "bias"),
                       (lambda: ops.route_topk_backward(x, x, pos), "grad"), (lambda: ops.expert_plan(pos[0], 3), "tokens, k"),
                       (lambda: ops.expert_plan(pos, 0), "positive"), (lambda: ops.expert_plan(pos + 0.5, 3), "whole"),
                       (lambda: ops.dispatch(x, pos.astype(np.float32)), "whole"), (lambda: ops.dispatch(x[:3], pos), "x must"),
                       (lambda: ops.combine(x, pos[:3]), "rows must"), (lambda: ops.combine(np.zeros((8, 3)), pos, np.zeros((4, 3))), "weights"),
                       (lambda: ops.combine_backward(x, np.zeros((8, 3)), pos), "grad"),
                       (lambda: ops.segment_mm_backward(x, x, np.zeros((2, 8, 8)), [1, 4]), "sum to"),
                       (lambda: ops.segment_mm_backward(x, x, np.zeros((2, 8, 8)), [4]), "one entry"),
                       (lambda: ops.segment_mm_backward(x, x, np.zeros((2, 7, 8)), [2, 2]), "inner")):
        with pytest.raises(DGLError, match=says):
            call()


def test_c_entry_points_check_their_arguments(lib):
    null, one = None, ctypes.c_void_p(16)
    assert lib.bgl_layer_norm(null, null, null, 2, 2, 1e-5, null, null, null, 0, 0, null) == INVALID
    assert lib.bgl_layer_norm(one, null, null, 2, 2, -1.0, one, null, null, 0, 0, null) == INVALID
    assert lib.bgl_layer_norm(one, null, null, 2, 2, 1e-5, one, null, null, 0, 2, null) == UNSUPPORTED
    assert lib.bgl_layer_norm(one, null, null, 2, 2, 1e-5, one, null, null, 9, 9, null) == UNSUPPORTED
    assert lib.bgl_layer_norm(null, null, null, 0, 2, 1e-5, null, null, null, 0, 0, null) == 0
    assert lib.bgl_layer_norm_backward(one, one, one, one, one, 2, 2, one, one, one, 0, 0, null, 0, null) == WORKSPACE
    assert lib.bgl_layer_norm_backward(null, one, one, one, one, 2, 2, one, null, null, 0, 0, null, 0, null) == INVALID
    route = lambda t, e, k, s, g, tg, top, dt: lib.bgl_route_topk(  # noqa: E731
        null, null, t, e, k, s, g, tg, top, 1, 1.0, null, null, dt, null)
    assert route(4, 8, 2, 0, 1, 1, 1, 0) == INVALID and b"null" in lib.bgl_last_error()
    assert route(4, 8, 2, 0, 1, 1, 1, 1) == UNSUPPORTED  # float64 logits
    assert route(4, 8, 2, 5, 1, 1, 1, 0) == INVALID and route(4, 8, 0, 0, 1, 1, 1, 0) == INVALID
    assert route(4, 8, 2, 0, 3, 1, 1, 0) == INVALID and route(4, 8, 2, 0, 2, 3, 1, 0) == INVALID
    assert route(4, 8, 5, 0, 2, 1, 1, 0) == INVALID and route(4, 8, 2, 0, 2, 1, 3, 0) == INVALID
    assert route(4, 2000, 2, 0, 1, 1, 1, 0) == UNSUPPORTED and route(4, 99, 33, 0, 1, 1, 1, 0) == UNSUPPORTED
    assert route(4, 66, 2, 0, 33, 1, 1, 0) == UNSUPPORTED and route(0, 8, 2, 0, 1, 1, 1, 0) == 0
    assert lib.bgl_route_topk_backward(null, null, null, 4, 8, 2, 0, 1, 1.0, null, 0, null) == INVALID
    assert lib.bgl_expert_plan(null, 4, 0, one, one, null, 0, null) == INVALID
    assert lib.bgl_expert_plan(one, 4, 8192, one, one, null, 0, null) == UNSUPPORTED
    assert lib.bgl_expert_plan(one, 1 << 31, 4, one, one, null, 0, null) == UNSUPPORTED
    assert lib.bgl_expert_plan(one, 1 << 20, 4, one, one, null, 0, null) == WORKSPACE
    assert lib.bgl_dispatch_rows(null, null, 4, 2, 8, null, 0, null) == INVALID
    assert lib.bgl_dispatch_rows(one, one, 1 << 30, 2, 8, one, 0, null) == UNSUPPORTED
    assert lib.bgl_combine_rows(null, null, null, 4, 2, 8, null, 0, null) == INVALID
    assert lib.bgl_combine_rows(one, one, null, 4, 2, 8, one, 7, null) == UNSUPPORTED
    assert lib.bgl_combine_rows_backward(null, null, null, null, 4, 2, 8, null, null, 0, null) == INVALID
    grad = lambda n, d1, r, d2, ws, dt=0: lib.bgl_segment_mm_backward(  # noqa: E731
        one, one, one, one, n, d1, r, d2, one, one, dt, null, ws, null)
    assert grad(-1, 2, 2, 2, 0) == INVALID and grad(2, 2, 2, 2, 0, 9) == UNSUPPORTED and grad(2, 2, 2, 2, 0) == WORKSPACE
    assert grad(2, 1 << 23, 2, 2, 0) == UNSUPPORTED
    assert lib.bgl_segment_mm_backward(one, one, one, null, 2, 2, 2, 2, one, one, 0, null, 0, null) == INVALID


def test_workspace_sizes(lib):
    assert lib.bgl_expert_plan_workspace_size(100, 8) == 0  # one launch, no workspace
    assert lib.bgl_expert_plan_workspace_size(1 << 20, 64) > 0
    assert lib.bgl_layer_norm_backward_workspace_size(0, 8, 0) >= 0
    assert lib.bgl_layer_norm_backward_workspace_size(1000, 4096, 2) >= 2 * 4096 * 4
    small = lib.bgl_segment_mm_backward_workspace_size(100, 64, 8, 64, 2)
    large = lib.bgl_segment_mm_backward_workspace_size(1 << 20, 2048, 8, 2048, 2)
    # the partial tiles: at most four 256 x 256 float32 tiles a CTA of a 148-SM device, none below 256 rows
    assert small < 1 << 16 and large < 148 * 4 * 256 * 256 * 4 + (1 << 20)
