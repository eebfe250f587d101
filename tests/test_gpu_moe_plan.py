"""The expert plan where its counters fill a block's shared memory, and positions
that are wider than its own."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import mojodgl.ops as ops  # noqa: E402


# the largest counts of 8 to 2 warps' counters in 48 KB with the warps' sums beside them, and
# those around: at 12288 / warps counters the sums have no room left
@pytest.mark.parametrize("experts", [1530, 1531, 1532, 1535, 1536, 1749, 1750, 1754, 1755, 2041, 2042, 2047, 2048, 2450, 2451, 2456,
                                     2457, 3063, 3064, 3071, 4084, 4085, 4095, 4096, 6127, 6128, 6143, 6144, 8190, 8191])
def test_plan_at_every_number_of_warps(experts):
    g = torch.Generator(device="cuda").manual_seed(experts)
    for tokens, k in ((0, 2), (5, 2), (700, 1), (20000, 3)):  # one chunk, and several
        idx = torch.randint(-1, experts + 1, (tokens, k), device="cuda", generator=g)
        plan = ops.expert_plan(idx, experts)
        flat = idx.reshape(-1).cpu().numpy()
        bins = np.where((flat < 0) | (flat >= experts), experts, flat)
        place = np.empty(len(flat), dtype=np.int64)
        place[np.argsort(bins, kind="stable")] = np.arange(len(flat))
        np.testing.assert_array_equal(plan.counts.cpu().numpy(), np.bincount(bins, minlength=experts + 1)[:experts])
        np.testing.assert_array_equal(plan.positions.cpu().numpy().reshape(-1), np.where(bins == experts, ~place, place))


def test_wide_positions_that_no_plan_gives_are_skipped():
    """64-bit positions beyond 32 bits are outside the rows, not their low halves."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x, rows, w = (torch.randn(*s, device="cuda", generator=g) for s in ((4, 16), (8, 16), (4, 2)))
    bad = torch.tensor([[1 << 32, (1 << 32) + 7], [-(1 << 32), -(1 << 33) - 3], [0, 1], [2, 3]], device="cuda")
    for pos in (bad, bad.cpu().numpy()):
        give = (lambda t: t) if isinstance(pos, torch.Tensor) else (lambda t: t.cpu().numpy())
        y = torch.as_tensor(ops.combine(give(rows), pos, give(w))).cuda()
        assert not y[:2].any() and torch.equal(y[2:], ops.combine(rows[:4], torch.arange(4, device="cuda").view(2, 2), w[2:]))
        drows, dw = (torch.as_tensor(t).cuda() for t in ops.combine_backward(give(x), give(rows), pos, give(w)))
        assert not dw[:2].any() and torch.equal(drows[0], w[2, 0] * x[2]) and torch.equal(drows[3], w[3, 1] * x[3])
        sent = torch.as_tensor(ops.dispatch(give(x), pos)).cuda()
        assert torch.equal(sent[:4], x[[2, 2, 3, 3]])
    wide = np.array([[1 << 32, 0], [(1 << 32) + 1, 1], [2, 3], [4, 5]], dtype=np.uint64)
    assert torch.equal(torch.as_tensor(ops.combine(rows.cpu().numpy(), wide)[0]).cuda(), rows[0])
