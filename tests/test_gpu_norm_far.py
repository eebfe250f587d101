"""Layer norm of rows whose spread is small beside their mean.

u = 2^-24 (2^-53 for float64).  With m the most additions between a value and a
sum of d of them (the values of a thread, its warp, its block), a mean is off by
E = m u |mean| at most.  x - mean is then exact (the two are within a factor of
two), and what the mean is off by is the mean of those differences, known to
m u (E + s) for a spread of s.  So a result is off by m u (E + s) rstd, and by
its relative error of the spread, m u (s^2 + 3 E^2 + 2 E s) rstd^2, beside its own
roundings.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

import mojodgl.ops as ops  # noqa: E402

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -24, torch.float64: 2.0 ** -53}
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float64: 2.0 ** -53}


def check(x, eps=1e-5):
    d, u = x.shape[-1], UNIT[x.dtype]
    m = 16 + 5 + 16 + 4 + d // 256  # values of a thread, warps, and the roundings around them
    g = torch.Generator(device="cuda").manual_seed(d)
    w, b = (torch.randn(d, device="cuda", generator=g, dtype=torch.float64).to(x.dtype) for _ in range(2))
    y, mean, rstd = ops.layer_norm(x, w, b, eps=eps, return_stats=True)
    xd, wd, bd = x.double(), w.double(), b.double()
    mu = xd.mean(-1, keepdim=True)
    s = (xd - mu).square().mean(-1, keepdim=True).sqrt()
    if x.dtype == torch.float64:  # the reference's own mean is off as much
        mu, s = (xd - xd[:, :1]).mean(-1, keepdim=True) + xd[:, :1], (xd - xd[:, :1]).std(-1, correction=0, keepdim=True)
    rs = 1 / (s * s + eps).sqrt()
    xhat = (xd - mu) * rs
    want = xhat * wd + bd
    far = m * u * mu.abs()
    spread = m * u * (s * s + 3 * far * far + 2 * far * s) * rs * rs
    tol = (m * u * (far + s) * rs + xhat.abs() * (spread + 4 * u)) * wd.abs() + 4 * u * (xhat * wd).abs() + 4 * u * bd.abs()
    if x.dtype == torch.float64:
        tol = tol + 4 * u * (mu.abs() * rs) * wd.abs()  # mu's own rounding in the reference
    tol = tol + ROUND[x.dtype] * want.abs()
    err = (y.double() - want).abs()
    assert (err <= tol).all(), (float((err - tol).max()), float(err.max()))
    assert ((mean.double() - mu[..., 0]).abs() <= 2 * u * mu[..., 0].abs() + 2 * m * u * (far + s)[..., 0]).all()
    assert ((rstd.double() - rs[..., 0]).abs() <= (spread[..., 0] + 8 * u) * rs[..., 0]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("d", [3, 33, 96, 257, 1000, 1001, 2047, 4100, 8000, 20001, 70000])
def test_constant_rows_of_any_size_give_the_bias(dtype, d):
    values = torch.tensor([0.1, 1000.1, -12345.678, 1e5, -3e7], device="cuda", dtype=torch.float64).to(dtype)
    check(values[:, None].expand(5, d).contiguous())


@pytest.mark.parametrize("d", [33, 256, 777, 1000, 4096, 7001, 20001, 70000])
def test_rows_far_from_zero(d):
    g = torch.Generator(device="cuda").manual_seed(d)
    x = torch.randn(9, d, device="cuda", generator=g)
    for far in (3e3, 1e5, 1e6):
        check(x + far)
        check(-far + x * 30)
    flat = torch.empty(9 * d + 1, device="cuda")
    flat[1:] = (x + 1e5).view(-1)
    check(flat[1:].view(9, d))  # rows that do not begin on 16 bytes
