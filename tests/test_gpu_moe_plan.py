"""The expert plan where its counters fill a block's shared memory."""

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
