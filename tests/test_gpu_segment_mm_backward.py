"""segment_mm's gradients against float64 products, segment by segment.

Tolerance: a float32 (float64) sum of n terms in any order is off by at most
n u times the sum of their magnitudes, u = 2^-24 (2^-53); bfloat16 operands
multiply exactly and their float32 sums may drop bits below the last one of the
larger summand at every step (2 u a term).  What is rounded to bfloat16 gets
2^-8 of its value on top.
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import mojodgl.ops as ops  # noqa: E402
from mojodgl import _lib  # noqa: E402
from mojodgl.base import DGLError  # noqa: E402

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -23, torch.float64: 2.0 ** -53}
ROUND = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float64: 0.0}
TYPES = [torch.float32, torch.bfloat16, torch.float64]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype):
    return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float64).to(dtype)


def lengths(seed, n, r, zero=()):
    rng = np.random.default_rng(seed)
    seglen = rng.multinomial(n, rng.dirichlet(0.7 * np.ones(r)))
    for z in zero:
        seglen[(z + 1) % r] += seglen[z]
        seglen[z] = 0
    return seglen


def reference(grad, a, b, seglen):
    """da, db and the sums of the magnitudes of their terms, in float64."""
    g, x, w = grad.double(), a.double(), b.double()
    da, sa = torch.zeros_like(x), torch.zeros_like(x)
    db, sb = torch.zeros_like(w), torch.zeros_like(w)
    start = 0
    for r, n in enumerate(int(v) for v in seglen):
        rows = slice(start, start + n)
        da[rows], sa[rows] = g[rows] @ w[r].T, g[rows].abs() @ w[r].abs().T
        db[r], sb[r] = x[rows].T @ g[rows], x[rows].abs().T @ g[rows].abs()
        start += n
    return da, sa, db, sb


def check(grad, a, b, seglen):
    da, db = ops.segment_mm_backward(grad, a, b, seglen)
    assert _lib.lib().bgl_tc_error() == 0
    ra, sa, rb, sb = reference(grad, a, b, seglen)
    u, rnd = UNIT[a.dtype], ROUND[a.dtype]
    assert da.dtype == db.dtype == a.dtype and da.shape == a.shape and db.shape == b.shape
    err, tol = (da.double() - ra).abs(), (b.shape[2] + 4) * u * sa + rnd * ra.abs()
    assert (err <= tol).all(), float((err - tol).max())
    longest = max([int(v) for v in seglen], default=0)
    err, tol = (db.double() - rb).abs(), (longest + 4) * u * sb + rnd * rb.abs()
    assert (err <= tol).all(), float((err - tol).max())
    return da, db


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,r,d1,d2", [(1, 1, 1, 1), (5, 3, 2, 3), (70, 4, 8, 8), (190, 8, 64, 40), (300, 3, 33, 65), (513, 2, 128, 256),
                                       (640, 5, 72, 136), (1000, 7, 256, 256), (900, 40, 24, 16), (2000, 3, 264, 520), (129, 1, 512, 128),
                                       (260, 2, 1032, 16), (77, 2, 16, 1024), (3000, 1, 136, 136), (64, 64, 96, 96)])
def test_sizes(dtype, n, r, d1, d2):
    g = gen(n + r + d1 + d2)
    seglen = lengths(n, n, r, zero=(r // 2,) if r > 1 else ())
    check(randn(g, n, d2, dtype=dtype), randn(g, n, d1, dtype=dtype), randn(g, r, d1, d2, dtype=dtype), seglen)


@pytest.mark.parametrize("dtype", TYPES)
def test_every_short_segment(dtype):
    """Segments of 0 to 140 rows, so every remainder of a tile occurs."""
    g = gen(4)
    seglen = np.arange(141)
    n = int(seglen.sum())
    check(randn(g, n, 64, dtype=dtype), randn(g, n, 128, dtype=dtype), randn(g, 141, 128, 64, dtype=dtype), seglen)


@pytest.mark.parametrize("d1,d2", [(64, 72), (256, 256), (320, 8)])
def test_sums_of_a_few_rows_one_after_another(d1, d2):
    """Hundreds of sums of 1 to 130 rows a worker: several parts of a slice are under way at once."""
    r = 6000
    seglen = np.random.default_rng(31).integers(1, 131, r)
    seglen[:5] = 1
    seglen[-100:] = 3
    n = int(seglen.sum())
    g = gen(32)
    grad, a, b = randn(g, n, d2, dtype=torch.bfloat16), randn(g, n, d1, dtype=torch.bfloat16), randn(g, r, d1, d2, dtype=torch.bfloat16)
    none, db = ops.segment_mm_backward(grad, a, b, seglen, need_a=False)
    assert none is None and _lib.lib().bgl_tc_error() == 0
    da, none = ops.segment_mm_backward(grad, a, b, seglen, need_b=False)
    assert none is None and _lib.lib().bgl_tc_error() == 0
    both = ops.segment_mm_backward(grad, a, b, seglen)
    assert _lib.lib().bgl_tc_error() == 0
    assert torch.equal(da, both[0]) and torch.equal(db, both[1])
    some = np.r_[0:40, r - 140:r - 80]  # these against float64
    first = np.concatenate([[0], np.cumsum(seglen)])
    at = torch.as_tensor(np.concatenate([np.arange(first[k], first[k + 1]) for k in some]), device="cuda")
    ra, sa, rb, sb = reference(grad[at], a[at], b[torch.as_tensor(some, device="cuda")], seglen[some])
    u, rnd = UNIT[torch.bfloat16], ROUND[torch.bfloat16]
    assert bool(((da[at].double() - ra).abs() <= (d2 + 4) * u * sa + rnd * ra.abs()).all())
    terms = torch.as_tensor(seglen[some], device="cuda").view(-1, 1, 1)
    got = db[torch.as_tensor(some, device="cuda")].double()
    assert bool(((got - rb).abs() <= (terms + 4) * u * sb + rnd * rb.abs()).all())


@pytest.mark.parametrize("d1,d2", [(16, 8), (128, 16), (8, 264), (264, 8), (16, 2048)])
def test_narrow_blocks_and_long_sums(d1, d2):
    """Blocks that one of two workers has no values of, over hundreds of slices."""
    seglen = np.array([20000, 0, 7001, 13])
    n = int(seglen.sum())
    g = gen(33)
    check(randn(g, n, d2, dtype=torch.bfloat16), randn(g, n, d1, dtype=torch.bfloat16), randn(g, 4, d1, d2, dtype=torch.bfloat16), seglen)


@pytest.mark.parametrize("n,r,d1,d2", [(70000, 9, 256, 256), (70001, 300, 200, 256), (141000, 64, 72, 128), (66001, 1, 8, 256), (300007, 1200, 256, 64)])
def test_blocks_of_one_tile_and_many_rows(n, r, d1, d2):
    """Segments end everywhere in a tile, the last rows belong to none."""
    g = gen(34 + d1)
    seglen = lengths(n, n - 37, r, zero=(r // 3,) if r > 1 else ())
    grad, a, b = randn(g, n, d2, dtype=torch.bfloat16), randn(g, n, d1, dtype=torch.bfloat16), randn(g, r, d1, d2, dtype=torch.bfloat16)
    first = check(grad, a, b, seglen)
    assert not first[0][-37:].any()
    again = ops.segment_mm_backward(grad, a, b, seglen)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_past_the_segments_and_empty_ones(dtype):
    g = gen(5)
    seglen = np.array([0, 100, 0, 0, 37, 0])
    n = 300
    grad, a, b = randn(g, n, 48, dtype=dtype), randn(g, n, 80, dtype=dtype), randn(g, 6, 80, 48, dtype=dtype)
    grad[137:], a[137:] = float("nan"), float("inf")  # rows of no segment
    da, db = ops.segment_mm_backward(grad, a, b, seglen)
    assert not da[137:].any() and not db[[0, 2, 3, 5]].any()
    ra, rb = ops.segment_mm_backward(grad[:137].clone(), a[:137].clone(), b, seglen)
    assert torch.equal(da[:137], ra) and torch.equal(db, rb)


@pytest.mark.parametrize("dtype", TYPES)
def test_not_a_number_stays_in_its_segment(dtype):
    g = gen(6)
    seglen = np.array([70, 1, 45, 130, 64])
    n = int(seglen.sum())
    grad, a, b = randn(g, n, 64, dtype=dtype), randn(g, n, 128, dtype=dtype), randn(g, 5, 128, 64, dtype=dtype)
    clean = ops.segment_mm_backward(grad, a, b, seglen)
    grad[70:71], a[75, 3], b[3, 5, 7] = float("nan"), float("inf"), float("nan")  # segments 1, 2 and 3
    da, db = ops.segment_mm_backward(grad, a, b, seglen)
    for r in (0, 3, 4):
        assert torch.equal(db[r], clean[1][r])
    assert db[1].isnan().all() and not db[2, 3].isfinite().any() and db[2, 4].isfinite().all()
    for rows in (slice(0, 70), slice(71, 116), slice(246, 310)):
        assert torch.equal(da[rows], clean[0][rows])
    assert da[70].isnan().all() and da[116:246, 5].isnan().all() and da[116:246, 6].isfinite().all()


def test_one_side_only_and_the_same_bits_again():
    g = gen(7)
    for dtype in TYPES:
        seglen = lengths(7, 4000, 6)
        grad, a, b = randn(g, 4000, 128, dtype=dtype), randn(g, 4000, 256, dtype=dtype), randn(g, 6, 256, 128, dtype=dtype)
        da, db = check(grad, a, b, seglen)
        for dev in (torch.from_numpy(seglen).cuda(), torch.from_numpy(seglen)):
            assert torch.equal(ops.segment_mm_backward(grad, a, b, dev, need_b=False)[0], da)
            none, again = ops.segment_mm_backward(grad, a, b, dev, need_a=False)
            assert none is None and torch.equal(again, db)


def test_lengths_on_the_device_are_clamped():
    g = gen(8)
    grad, a, b = randn(g, 100, 32, dtype=torch.bfloat16), randn(g, 100, 64, dtype=torch.bfloat16), randn(g, 3, 64, 32, dtype=torch.bfloat16)
    got = ops.segment_mm_backward(grad, a, b, torch.tensor([40, -7, 1 << 40], device="cuda"))
    want = ops.segment_mm_backward(grad, a, b, np.array([40, 0, 60]))
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dtype", TYPES)
def test_empty(dtype):
    def z(*shape):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    da, db = ops.segment_mm_backward(z(0, 8), z(0, 16), z(3, 16, 8) + 1, np.zeros(3, int))
    assert da.shape == (0, 16) and db.shape == (3, 16, 8) and not db.any()
    da, db = ops.segment_mm_backward(z(9, 8) + 1, z(9, 16), z(0, 16, 8), np.zeros(0, int))
    assert not da.any() and db.shape == (0, 16, 8)
    da, db = ops.segment_mm_backward(z(9, 0), z(9, 16), z(2, 16, 0), np.array([4, 5]))
    assert not da.any() and db.shape == (2, 16, 0)
    da, db = ops.segment_mm_backward(z(9, 8), z(9, 0), z(2, 0, 8), np.array([4, 5]))
    assert da.shape == (9, 0) and db.shape == (2, 0, 8)


def test_strides_and_alignment():
    g = gen(9)
    seglen = np.array([50, 30, 20])
    for dtype in (torch.bfloat16, torch.float32):
        wide, b = randn(g, 100, 300, dtype=dtype), randn(g, 3, 128, 64, dtype=dtype)
        for grad, a in ((wide[:, 1:65], wide[:, 70:198]), (wide.t()[:100, :64], wide[:, 2:258:2]),
                        (wide[:1, :64].expand(100, 64), wide[:, :128])):
            got = ops.segment_mm_backward(grad, a, b.transpose(1, 2).contiguous().transpose(1, 2), seglen)
            want = ops.segment_mm_backward(grad.clone(memory_format=torch.contiguous_format),
                                           a.clone(memory_format=torch.contiguous_format), b, seglen)
            assert all(torch.equal(p, q) for p, q in zip(got, want))
        flat = randn(g, 100 * 64 + 8, dtype=dtype)
        check(flat[1:1 + 6400].view(100, 64), wide[:, :128].contiguous(), b, seglen)
        flat_b = randn(g, 3 * 128 * 64 + 3, dtype=dtype)
        check(wide[:, :64].contiguous(), wide[:, :128].contiguous(), flat_b[3:].view(3, 128, 64), seglen)


def test_more_than_two_to_the_31_values():
    g = gen(10)
    n, d1, d2 = (1 << 21) + 77, 1024, 64
    seglen = np.array([n - 300, 300])
    a = torch.zeros(n, d1, dtype=torch.bfloat16, device="cuda")
    grad = torch.zeros(n, d2, dtype=torch.bfloat16, device="cuda")
    a[-400:], grad[-400:] = randn(g, 400, d1, dtype=torch.bfloat16), randn(g, 400, d2, dtype=torch.bfloat16)
    b = randn(g, 2, d1, d2, dtype=torch.bfloat16)
    da, db = ops.segment_mm_backward(grad, a, b, seglen)
    ra, sa, rb, sb = reference(grad[-400:], a[-400:], b, [100, 300])
    assert ((da[-400:].double() - ra).abs() <= 68 * 2.0 ** -23 * sa + 2.0 ** -8 * ra.abs()).all() and not da[:-400].any()
    assert ((db.double() - rb).abs() <= 304 * 2.0 ** -23 * sb + 2.0 ** -8 * rb.abs()).all()


def test_against_differences():
    """The gradients are the slopes of sum(grad * segment_mm(a, b)) in float64."""
    g = gen(11)
    seglen = np.array([3, 0, 4])
    a, b, grad = (randn(g, *s, dtype=torch.float64) for s in ((8, 3), (3, 3, 4), (8, 4)))
    for t, got in zip((a, b), ops.segment_mm_backward(grad, a, b, seglen)):
        for i in range(t.numel()):
            keep, value = float(t.view(-1)[i]), []
            for move in (1e-6, -1e-6):
                t.view(-1)[i] = keep + move
                value.append(float((ops.segment_mm(a, b, seglen) * grad).sum()))
            t.view(-1)[i] = keep
            assert abs((value[0] - value[1]) / 2e-6 - float(got.reshape(-1)[i])) < 1e-8  # linear: rounding only


def test_types_and_numpy():
    rng = np.random.default_rng(12)
    seglen = np.array([4, 6])
    a, b, grad = rng.normal(size=(10, 6)), rng.normal(size=(2, 6, 5)), rng.normal(size=(10, 5))
    da, db = ops.segment_mm_backward(grad, a, b, seglen)
    assert isinstance(da, np.ndarray) and da.dtype == np.float64
    np.testing.assert_allclose(da[4:], grad[4:] @ b[1].T, rtol=1e-12, atol=1e-13)
    np.testing.assert_allclose(db[0], a[:4].T @ grad[:4], rtol=1e-12, atol=1e-13)
    half = [torch.from_numpy(v).half().cuda() for v in (grad, a, b)]
    assert ops.segment_mm_backward(*half, seglen)[0].dtype == torch.float32


def test_refusals():
    a, b, grad = torch.zeros(10, 6, device="cuda"), torch.zeros(2, 6, 5, device="cuda"), torch.zeros(10, 5, device="cuda")
    for call in (lambda: ops.segment_mm_backward(grad, a, b, [4, 7]), lambda: ops.segment_mm_backward(grad, a, b, [-1, 7]),
                 lambda: ops.segment_mm_backward(grad, a, b, [4, 3, 3]), lambda: ops.segment_mm_backward(grad, a, b, [4.5, 5]),
                 lambda: ops.segment_mm_backward(grad[:9], a, b, [4, 6]), lambda: ops.segment_mm_backward(grad, a[:, :5], b, [4, 6]),
                 lambda: ops.segment_mm_backward(grad, a, b[0], [4, 6]), lambda: ops.segment_mm_backward(grad.to(torch.complex64), a, b, [4, 6])):
        with pytest.raises(DGLError):
            call()
