"""Layer norm, forward and backward, against the formula in 64 bits.

Tolerances come from the usual bound on a floating sum: n terms summed in any
order are off by at most n * u * (sum of their magnitudes), u = 2^-24 for
float32 sums and 2^-53 for float64.  A result rounded to bfloat16 is off by
another 2^-8 of its value (half a step is 2^-9; one more for what crosses a
rounding boundary).
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import mojodgl.ops as ops  # noqa: E402
from mojodgl.base import DGLError  # noqa: E402

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -24, torch.float64: 2.0 ** -53}
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float64: 2.0 ** -53}
TYPES = [torch.float32, torch.bfloat16, torch.float64]


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float64).to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def check(got, ref, tol):
    err = (got.double() - ref).abs()
    bad = err > tol
    assert not bad.any(), "max excess {}".format(float((err - tol).max()))


def forward_reference(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + eps)
    y = (x - mean) * rstd
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, mean[..., 0], rstd[..., 0]


def check_forward(x, w, b, eps=1e-5):
    y, mean, rstd = ops.layer_norm(x, w, b, eps=eps, return_stats=True)
    ry, rm, rr = forward_reference(x, w, b, eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    d, u = x.shape[-1], UNIT[x.dtype]
    n = d + 16  # terms of a sum, and the roundings around it
    xd = x.double().abs()
    check(mean, rm, n * u * xd.mean(-1))
    # a centred value is off by n u (|x| + mean |x|), in units of the row's spread
    off = n * u * ((xd + xd.mean(-1, keepdim=True)) * rr[..., None])
    worst = off.square().mean(-1).sqrt()  # relative error of the spread that this makes
    check(rstd, rr, rr * (worst + n * u))
    ww = 1.0 if w is None else w.double().abs()
    bb = 0.0 if b is None else b.double().abs()
    xhat = ((x.double() - rm[..., None]) * rr[..., None]).abs()
    tol = (off + xhat * (worst[..., None] + n * u)) * ww + 4 * u * (xhat * ww + bb) + ROUND[x.dtype] * ry.abs()
    check(y, ry, tol)
    assert torch.equal(y, ops.layer_norm(x, w, b, eps=eps))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (1, 7), (5, 31), (2, 32), (7, 33), (4, 255), (3, 256),
                                    (2, 1000), (1, 2048), (3, 4096), (2, 8192), (2, 8200), (3, 20001), (1, 70000),
                                    (1500, 40), (3000, 520)])
def test_forward_sizes(dtype, rows, d):
    g = gen(rows * 100003 + d)
    x = randn(g, rows, d, dtype=dtype) + 0.5
    w, b = randn(g, d, dtype=dtype), randn(g, d, dtype=dtype)
    check_forward(x, w, b)
    check_forward(x, w, None)
    check_forward(x, None, None)


def test_forward_offset_and_scale():
    """A mean far from zero costs digits of x, not of the sums of squares."""
    g = gen(3)
    x = (randn(g, 40, 777) + 3000.0).float()
    check_forward(x, torch.ones(777, device="cuda"), torch.zeros(777, device="cuda"))
    check_forward((randn(g, 40, 777) * 1e-4).float(), None, None, eps=0.0)
    check_forward((randn(g, 40, 1024) * 1e15).float(), None, None)


@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
def test_forward_bf16_rows_with_either_weight(wdtype):
    g = gen(5)
    x = randn(g, 6, 4, 640, dtype=torch.bfloat16)
    check_forward(x, randn(g, 640, dtype=wdtype), randn(g, 640, dtype=wdtype))


def test_constant_rows_give_the_bias():
    for dtype in TYPES:
        x = torch.full((3, 96), 2.5, dtype=dtype, device="cuda")
        b = torch.arange(96, device="cuda").to(dtype)
        assert torch.equal(ops.layer_norm(x, torch.ones_like(b), b), b.expand(3, 96))


def test_not_a_number_stays_in_its_row():
    g = gen(6)
    x = randn(g, 5, 300)
    clean = ops.layer_norm(x)
    x[2, 17] = float("nan")
    x[4, 299] = float("inf")
    y = ops.layer_norm(x)
    assert y[2].isnan().all() and y[4].isnan().any()
    for row in (0, 1, 3):
        assert torch.equal(y[row], clean[row])


def test_strides_and_alignment():
    g = gen(7)
    base = randn(g, 64, 515)
    w = randn(g, 600)
    for x in (base[:, 1:514], base[::2, :512], base.t(), base[:, :512][3:9], base.view(-1)[1:1 + 64 * 500].view(64, 500),
              base[:1, :].expand(9, 515)):
        d = x.shape[1]
        check_forward(x, w[1:1 + d], None)  # the weight is not 16-byte aligned either
    flat = randn(g, 3 * 520 + 8, dtype=torch.bfloat16)
    for shift in (1, 2, 3, 8):
        check_forward(flat[shift:shift + 3 * 520].view(3, 520), None, None)


def test_empty_and_numpy():
    assert ops.layer_norm(torch.zeros(0, 8, device="cuda")).shape == (0, 8)
    y, mean, rstd = ops.layer_norm(torch.zeros(2, 0, 8, device="cuda"), return_stats=True)
    assert y.shape == (2, 0, 8) and mean.shape == rstd.shape == (2, 0)
    dx, dw, db = ops.layer_norm_backward(torch.zeros(0, 8, device="cuda"), torch.zeros(0, 8, device="cuda"),
                                         torch.zeros(0, device="cuda"), torch.zeros(0, device="cuda"),
                                         torch.ones(8, device="cuda"))
    assert dx.shape == (0, 8) and not dw.any() and not db.any()
    x = np.random.default_rng(1).normal(size=(4, 50))
    got = ops.layer_norm(x)
    assert isinstance(got, np.ndarray) and got.dtype == np.float64
    np.testing.assert_allclose(got, (x - x.mean(1, keepdims=True)) / np.sqrt(x.var(1, keepdims=True) + 1e-5), rtol=1e-11, atol=1e-12)


def check_backward(x, dy, w):
    _, mean, rstd = ops.layer_norm(x, w, return_stats=True)
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w)
    xd, gd = x.double(), dy.double()
    m, r = mean.double()[..., None], rstd.double()[..., None]
    d, u = x.shape[-1], UNIT[x.dtype]
    xhat = (xd - m) * r
    size = (xd.abs() + m.abs()) * r  # magnitude of the terms of xhat
    v = gd if w is None else gd * w.double()
    ref = r * (v - v.mean(-1, keepdim=True) - xhat * (v * xhat).mean(-1, keepdim=True))
    scale = r * (v.abs() + v.abs().mean(-1, keepdim=True) + size * (v.abs() * size).mean(-1, keepdim=True))
    check(dx, ref, (d + 16) * u * scale + ROUND[x.dtype] * ref.abs())
    assert dx.dtype == x.dtype
    if w is None:
        assert dw is None and db is None
        return
    rows = xd.numel() // d
    flat = lambda t: t.reshape(rows, d)  # noqa: E731
    rw, rb = flat(gd * xhat).sum(0), flat(gd).sum(0)
    assert dw.dtype == db.dtype == w.dtype
    check(dw, rw, (rows + 16) * u * flat(gd.abs() * size).sum(0) + ROUND[w.dtype] * rw.abs())
    check(db, rb, (rows + 16) * u * flat(gd.abs()).sum(0) + ROUND[w.dtype] * rb.abs())
    again = ops.layer_norm_backward(dy, x, mean, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))  # fixed order of the sums


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (1, 7), (5, 31), (300, 33), (257, 64), (4, 255), (513, 256), (2, 1000),
                                    (1, 2048), (700, 4096), (300, 8192), (2, 8200), (3, 20001), (5000, 72), (20000, 24)])
def test_backward_sizes(dtype, rows, d):
    g = gen(rows * 7 + d)
    x, dy = randn(g, rows, d, dtype=dtype) + 0.25, randn(g, rows, d, dtype=dtype)
    check_backward(x, dy, randn(g, d, dtype=dtype))
    check_backward(x, dy, None)


def test_backward_mixed_types_and_strides():
    g = gen(11)
    x, dy = randn(g, 70, 328, dtype=torch.bfloat16), randn(g, 70, 328, dtype=torch.bfloat16)
    check_backward(x, dy, randn(g, 328))
    check_backward(x[:, 1:300], dy[:, 3:302], randn(g, 299))
    check_backward(x.view(7, 10, 328), dy.view(7, 10, 328), randn(g, 328))
    check_backward(randn(g, 90, 65).t(), randn(g, 1, 90).expand(65, 90), randn(g, 90))


def test_backward_against_differences():
    """The gradients are the slopes of sum(dy * y) in float64."""
    g = gen(13)
    x, dy, w, b = (randn(g, *s, dtype=torch.float64) for s in ((4, 9), (4, 9), (9,), (9,)))
    _, mean, rstd = ops.layer_norm(x, w, b, return_stats=True)
    got = ops.layer_norm_backward(dy, x, mean, rstd, w)
    step = 1e-5
    for grad, t in zip(got, (x, w, b)):
        for i in range(t.numel()):
            keep = float(t.view(-1)[i])
            t.view(-1)[i] = keep + step
            up = float((ops.layer_norm(x, w, b) * dy).sum())
            t.view(-1)[i] = keep - step
            down = float((ops.layer_norm(x, w, b) * dy).sum())
            t.view(-1)[i] = keep
            # central differences: step^2 / 6 of a third derivative of order 10, and 1e-16 * 30 / step of rounding
            assert abs((up - down) / (2 * step) - float(grad.reshape(-1)[i])) < 1e-7


def test_more_than_two_to_the_31_values():
    """The last rows of an array whose offsets need 64 bits."""
    rows, d = (1 << 21) + 5, 1032
    x = torch.zeros(rows, d, dtype=torch.bfloat16, device="cuda")
    dy = torch.zeros(rows, d, dtype=torch.bfloat16, device="cuda")
    g = gen(17)
    x[-3:], dy[-3:] = randn(g, 3, d, dtype=torch.bfloat16), randn(g, 3, d, dtype=torch.bfloat16)
    w = randn(g, d)
    y, mean, rstd = ops.layer_norm(x, w, return_stats=True)
    small = ops.layer_norm(x[-3:].clone(), w, return_stats=True)
    assert torch.equal(y[-3:], small[0]) and torch.equal(mean[-3:], small[1]) and torch.equal(rstd[-3:], small[2])
    del y
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w)
    sdx, sdw, sdb = ops.layer_norm_backward(dy[-3:].clone(), x[-3:].clone(), mean[-3:].clone(), rstd[-3:].clone(), w)
    assert torch.equal(dx[-3:], sdx)
    torch.testing.assert_close(dw, sdw, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(db, sdb, rtol=1e-5, atol=1e-5)


def test_runs_on_the_current_stream():
    g = gen(19)
    side = torch.cuda.Stream()
    x = torch.zeros(64, 1024, device="cuda")
    fresh = randn(g, 64, 1024)
    big = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(4):
            big = big @ big * 1e-2  # keeps the stream busy before x is ready
        x.copy_(fresh)
        y = ops.layer_norm(x)
    side.synchronize()
    assert torch.equal(y, ops.layer_norm(fresh))


def test_refusals():
    x = torch.zeros(4, 8, device="cuda")
    s = torch.zeros(4, device="cuda")
    for call in (lambda: ops.layer_norm(x, bias=torch.zeros(8, device="cuda")), lambda: ops.layer_norm(x, torch.zeros(7, device="cuda")),
                 lambda: ops.layer_norm(torch.zeros(4, 0, device="cuda")), lambda: ops.layer_norm(torch.zeros((), device="cuda")),
                 lambda: ops.layer_norm(x, eps=-1.0), lambda: ops.layer_norm(x, eps=float("nan")),
                 lambda: ops.layer_norm(x.to(torch.complex64)),
                 lambda: ops.layer_norm_backward(x[:3], x, s, s), lambda: ops.layer_norm_backward(x, x, s[:3], s),
                 lambda: ops.layer_norm_backward(x, x, s, s[:, None]), lambda: ops.layer_norm_backward(x, x, s, s, torch.zeros(4, device="cuda"))):
        with pytest.raises(DGLError):
            call()
