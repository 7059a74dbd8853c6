"""Controls on rows of logits: offsets of any kind."""
import numpy as np
import pytest
import torch

from speculate_common import controls, put

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offsets", [[0, 10, 3, -2 ** 31], [0, 10, 3, -2 ** 31, 12], [0, 3, -2 ** 31 + 2, 12], [5, -2 ** 31, 12, 0],
                                     [-2 ** 31, 12, 2 ** 31 - 1], [2 ** 31 - 1, -2 ** 31, 12], [4, 4, -1, 4, 12]])
@pytest.mark.parametrize("words", [1, 32])
def test_offsets_that_descend(offsets, words):
    """A row is left as it is, or is a sequence's whose two offsets hold it; its path ends with the sequence and the rows."""
    n, rows = 300, 12
    g = torch.Generator("cuda").manual_seed(1)
    logits = torch.randn(rows, n, generator=g, device="cuda")
    tokens = torch.arange(rows, dtype=torch.int32, device="cuda") + 20
    # every node's bits are all set: all of a sequence's tokens are on each path
    spec = dict(offsets=put(offsets), tokens=tokens, ancestors=torch.full((rows, words), -1, dtype=torch.int32, device="cuda"),
                presence=torch.full((len(offsets) - 1,), 8.0, device="cuda"))
    out = torch.full((rows, n), 7.0, device="cuda")
    controls(logits, n, out, spec, len(offsets) - 1)
    torch.cuda.synchronize()
    x, got = logits.cpu().numpy(), out.cpu().numpy()
    for t in range(rows):
        fits = [np.full(n, np.float32(7))]
        for first, end in zip(offsets, offsets[1:]):
            if first <= t < end:
                y = x[t].copy()
                y[20 + max(first, 0):20 + min(end, rows, max(first, 0) + 32 * words)] -= np.float32(8)
                fits.append(y)
        assert any(np.array_equal(got[t], y) for y in fits), t
