"""Controls on rows of logits: offsets of any kind, n-grams at their longest and in histories at theirs."""
import time

import numpy as np
import pytest
import torch

from speculate_common import controls, controls64, put

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


@pytest.mark.parametrize("ngram", [2, 3, 63, 64, 65, 66, 200, 65536, 2 ** 31 - 1])
def test_longest_ngrams(ngram):
    """More than 64 tokens are off."""
    n, rng = 40, np.random.default_rng(3)
    text = rng.integers(0, 4, 70).tolist()
    history = [text * 4, rng.integers(0, 2, 280).tolist(), [5] * 280, ([6] * 70 + [7]) * 3 + [6] * 67]
    logits = torch.randn(4, n, device="cuda")
    out = torch.zeros(4, n, device="cuda")
    controls(logits, n, out, dict(history=put(history), history_lengths=put([280] * 4), ngram=put([ngram] * 4)), 4)
    torch.cuda.synchronize()
    for t in range(4):
        want, _ = controls64(logits[t].double().cpu().numpy(), history[t], ngram=ngram if ngram <= 64 else 0)
        assert np.array_equal(out[t].double().cpu().numpy(), want), t


@pytest.mark.parametrize("ngram", [64, 65536])
def test_a_history_of_one_token(ngram):
    """Every place of the longest history fits an n-gram: 2^17 times 63 comparisons by one workgroup, some milliseconds."""
    n, width = 1000, 1 << 17
    logits = torch.randn(2, n, device="cuda")
    out = torch.zeros(2, n, device="cuda")
    history = torch.full((2, width), 3, dtype=torch.int32, device="cuda")
    history[1, 5::64] = 4  # every 64th another one: places that fit 62 tokens
    spec = dict(history=history, history_lengths=put([width, width]), ngram=put([ngram] * 2))
    controls(logits, n, out, spec, 2)
    torch.cuda.synchronize()
    begin = time.monotonic()
    controls(logits, n, out, spec, 2)
    torch.cuda.synchronize()
    assert time.monotonic() - begin < 1
    want = logits.clone()
    if ngram <= 64:
        want[0, 3] = float("-inf")
        want[1] = torch.from_numpy(controls64(logits[1].double().cpu().numpy(), history[1].tolist(), ngram=ngram)[0])
    assert torch.equal(out, want)
