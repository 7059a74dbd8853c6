"""Positions and ancestors of the nodes of drafted trees, node by node on the host."""
import numpy as np
import pytest
import torch

from speculate_common import paged_tree, put, random_parents, tree64

pytestmark = pytest.mark.gpu


def check(counts, words, window=0, pad=5, seed=0, parents=None, lengths=None):
    rng = np.random.default_rng(seed)
    offsets = np.concatenate([[0], np.cumsum(counts)]).tolist()
    tokens = offsets[-1] + pad
    if parents is None:
        parents = sum((random_parents(rng, c, 1 + seed % 7) for c in counts), [])
    parents = parents + [0] * pad
    lengths = [int(rng.integers(0, 1000)) + c for c in counts] if lengths is None else lengths
    want = tree64(lengths, offsets, parents, tokens, words, window)
    got = paged_tree(put(lengths), put(offsets), put(parents), tokens, words, window)
    for g, w in zip(got, want):
        assert np.array_equal(g.cpu().numpy(), w)


@pytest.mark.parametrize("words", [1, 2, 3, 8, 9, 16, 17, 32])
@pytest.mark.parametrize("window", [0, 1, 3, 40])
def test_random_trees(words, window):
    most = 32 * words
    check([1, most, 0, min(most, 33), most - 1, 2, min(most, 64)], words, window, seed=words)


@pytest.mark.parametrize("words", [1, 2, 5, 16, 32])
def test_chains_and_stars(words):
    n = 32 * words
    check([n, n], words, parents=list(range(-1, n - 1)) + [-1] + [0] * (n - 1))
    check([n, n], words, 7, parents=list(range(-1, n - 1)) + [-1] + [0] * (n - 1))


@pytest.mark.parametrize("words", [1, 4])
def test_parents_that_are_no_node_before(words):
    check([6, 4], words, parents=[-1, 1, 5, -7, 2 ** 31 - 1, 3, 0, 0, 2, 1])


@pytest.mark.parametrize("words", [1, 2, 6])
def test_too_many_nodes_and_short_lengths(words):
    """Such requests' tokens have no position; their neighbours' stay."""
    n = 32 * words
    check([3, n + 1, 4, 5, 200 + n], words, lengths=[10, 5000, 3, 5, 5000])


@pytest.mark.parametrize("words", [1, 2, 6])
def test_extreme_lengths(words):
    check([3, 4, 2, 1], words, lengths=[-2 ** 31, -2 ** 31 + 3, 2 ** 31 - 1, 1])


@pytest.mark.parametrize("rows", [1, 4, 5, 1000])
def test_many_requests(rows):
    check([(r * 7) % 20 for r in range(rows)], 1, seed=rows, pad=1000)
    check([(r * 7) % 90 for r in range(rows)], 3, seed=rows, pad=1)


def test_offsets_that_are_none():
    """Requests of offsets outside the step, or that descend, have no nodes; nothing outside is touched."""
    guard = torch.full((40,), -77, dtype=torch.int32, device="cuda")
    positions, ancestors = guard[8:18], torch.full((10, 1), -77, dtype=torch.int32, device="cuda")
    offsets = put([0, 3, -4, 5, 2 ** 31 - 1])
    paged_tree(put([10, 10, 10, 10]), offsets, put([-1, 0, 1] + [0] * 7), 10, 1, positions=positions, ancestors=ancestors)
    torch.cuda.synchronize()
    assert positions[:3].tolist() == [7, 8, 9] and ancestors[:3, 0].tolist() == [1, 3, 7]
    assert torch.all(guard[:8] == -77) and torch.all(guard[18:] == -77)


def test_no_tokens():
    paged_tree(put([5]), put([0, 0]), None, 0, 1, positions=torch.zeros(1, device="cuda"), ancestors=torch.zeros(1, device="cuda"))
    torch.cuda.synchronize()
