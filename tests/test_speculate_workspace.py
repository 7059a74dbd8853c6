"""Workspaces of the attention of several new tokens a request: sizes (no GPU is needed)."""
import itertools

import pytest

from plamo_hip import native


@pytest.mark.parametrize("heads,kv,dim", [(16, 1, 128), (32, 8, 64), (8, 2, 256), (7, 1, 64), (1, 1, 128), (4096, 256, 64)])
def test_enough_for_smaller_calls(heads, kv, dim):
    """A server allocates once, for the most rows and tokens that it will have."""
    size = native.load().plamo_kernel_attention_paged_tree_workspace
    rows, tokens = [1, 2, 3, 8, 32, 64, 65, 1000, 1025, 1 << 20], [0, 1, 2, 5, 24, 64, 73, 500, 4096, 1 << 20]
    sizes = {(r, t): size(r, t, heads, kv, dim) for r in rows for t in tokens}
    for (r, t), (r2, t2) in itertools.product(sizes, sizes):
        if r2 <= r and t2 <= t:
            assert sizes[r2, t2] <= sizes[r, t], (r2, t2, r, t)
