"""The workspace of segment_mm's gradients: offsets of each segment, and float32
partial tiles of 512 x 256 for the sums that are cut (at most three a pair of CTAs,
none where no sum has more than eight slices of 64 rows)."""

import pytest

from mojodgl import _lib

BF16, TILE, PAIRS = 2, 512 * 256 * 4, 148 // 2


def offsets(r):
    """Five arrays of r + 1 64-bit numbers, one of r 32-bit ones, five numbers; each
    on a 256-byte boundary, and the workspace brought to one."""
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    return 5 * up(8 * (r + 1)) + up(4 * r) + up(40) + 256


@pytest.mark.parametrize("d1,d2", [(8, 8), (256, 256), (520, 264), (2048, 2048)])
@pytest.mark.parametrize("r", [1, 8, 300])
def test_partial_tiles_only_where_a_sum_may_be_cut(d1, d2, r):
    size = lambda n: _lib.lib().bgl_segment_mm_backward_workspace_size(n, d1, r, d2, BF16)  # noqa: E731
    fixed = offsets(r)
    for n in (0, 1, 64, 190, 511, 512):
        assert size(n) <= fixed
    tiles = -(-d1 // 512) * -(-d2 // 256)
    for n in (513, 1024, 1025, 5000, 70000, 1 << 20):
        # a sum of L > 8 slices has at most ceil(L / 8) pieces
        assert size(n) >= min(2 * tiles, PAIRS) * TILE
        assert size(n) <= fixed + min(tiles * 2 * (n // 64) // 8, 3 * PAIRS) * TILE
    for dtype in (0, 1):
        assert _lib.lib().bgl_segment_mm_backward_workspace_size(1 << 20, d1, r, d2, dtype) <= fixed
