"""The paths that drawn tokens agree with, one request after the other on the host: kept tokens, lengths, pages given back,
moves, and calls that change nothing."""
import numpy as np
import pytest
import torch

from paged_common import make_tables
from speculate_common import ACCEPTED, accept_step, paged_accept, put, random_parents

pytestmark = pytest.mark.gpu


def build(counts, before, page, nodes, seed=0, agree=0.7, given=None, words=30, spare=4):
    rng = np.random.default_rng(seed)
    offsets = np.concatenate([[0], np.cumsum(counts)]).tolist()
    total = offsets[-1]
    parents = sum((random_parents(rng, c) for c in counts), [])
    # few different tokens, so that siblings agree too
    tokens, drawn = rng.integers(0, words, total).tolist(), rng.integers(0, words, total).tolist()
    for r, first in enumerate(offsets[:-1]):
        for i in range(counts[r]):
            if parents[first + i] >= 0 and rng.random() < agree:
                drawn[first + parents[first + i]] = tokens[first + i]
    lengths = [b + c for b, c in zip(before, counts)]
    held = [-(-n // page) for n in lengths]
    pages = sum(held) + spare
    tables = make_tables(rng, lengths, page, pages, max(1, max(held)))
    used = set(tables[tables >= 0].tolist())
    free = [p for p in range(pages) if p not in used][:spare]
    return dict(lengths=lengths, offsets=offsets, parents=parents, tokens=tokens, drawn=drawn,
                given=[1] * len(counts) if given is None else given, tables=tables.tolist(), free=free), pages


def check(case, pages, page, nodes, given=True):
    want_free = list(case["free"])
    want = accept_step(case["lengths"], case["offsets"], case["parents"], case["tokens"], case["drawn"], case["given"],
                       case["tables"], page, want_free, pages, nodes)
    rows = len(case["lengths"])
    s = {k: put(v) for k, v in case.items() if k not in ("free", "given")}
    if given:
        s["given"] = put(case["given"])
    stack = np.full(pages, -5)
    stack[:len(case["free"])] = case["free"]
    s.update(free=put(stack), free_count=put([len(case["free"])]), lengths_out=put([-9] * rows), free_out=put([-9]),
             accepted=put(np.full((rows, nodes + 1), -9)), accepted_counts=put([-9] * rows), last=put([-9] * rows),
             status=put([-9]), **{k: put(np.full((rows, nodes), -9)) for k in ("from", "to")})
    paged_accept(s, page, nodes, pages)
    torch.cuda.synchronize()
    for name in ACCEPTED:
        got = s[name].cpu().numpy()
        assert np.array_equal(got.reshape(-1), np.array(want[name], dtype=np.int32).reshape(-1)), (name, got, want[name])
    assert s["free"].tolist()[:len(want_free)] == want_free and torch.all(s["free"][len(want_free):] == -5)
    assert np.array_equal(s["tables"].cpu().numpy(), np.array(case["tables"]))
    return want


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("page", [1, 3, 16, 64])
def test_random_trees(page, seed):
    rng = np.random.default_rng(seed)
    counts = rng.integers(0, 12, 9).tolist()
    case, pages = build(counts, rng.integers(0, 70, 9).tolist(), page, 12, seed)
    assert check(case, pages, page, 12)["status"] == 0


@pytest.mark.parametrize("count", [1, 2, 63, 64, 65, 66, 128, 129, 300])
def test_numbers_of_nodes(count):
    case, pages = build([count, 3, count], [20, 0, 31], 8, 300, count, agree=0.9)
    check(case, pages, 8, 300)


def test_whole_chains_and_nothing_kept():
    n = 100
    case, pages = build([n, n], [5, 6], 4, n, spare=0)
    case["parents"] = list(range(-1, n - 1)) * 2
    case["tokens"] = list(range(2 * n))
    case["drawn"] = [t + 1 for t in range(n)] + [500] * n
    want = check(case, pages, 4, n)
    assert want["accepted_counts"] == [n, 1] and want["lengths_out"] == [n + 5, 7]


def test_given_tokens():
    case, pages = build([20, 5, 1, 8, 0], [3, 9, 0, 40, 7], 16, 20, 3, given=[20, 2, 1, 0, 5])
    check(case, pages, 16, 20)
    case["given"] = [99, -3, 0, 8, 1]
    check(case, pages, 16, 20)
    case["given"] = [1] * 5
    check(case, pages, 16, 20, given=False)


def test_siblings_of_one_token():
    """The first of nodes that agree."""
    case, pages = build([6], [10], 16, 6)
    case.update(parents=[-1, 0, 0, 0, 2, 1], tokens=[9, 4, 4, 4, 7, 7], drawn=[4, 7, 7, 7, 1, 2])
    want = check(case, pages, 16, 6)
    assert want["accepted"] == [[4, 7, 2, -1, -1, -1, -1]]


def test_tokens_that_none_was_drawn_of():
    case, pages = build([4, 4], [10, 3], 16, 4)
    case.update(parents=[-1, 0, 1, 2] * 2, tokens=[5, -1, 3, 3, 5, 6, 3, 3], drawn=[-1, 3, 3, 3, 6, -1, 3, 3])
    want = check(case, pages, 16, 4)
    assert want["accepted"] == [[-1] * 5, [6, -1, -1, -1, -1]] and want["accepted_counts"] == [1, 2]


def test_parents_that_come_after():
    case, pages = build([5], [10], 16, 5)
    case.update(parents=[3, 0, 4, 1, 2 ** 31 - 1], tokens=[1] * 5, drawn=[1] * 5)
    check(case, pages, 16, 5)


def test_entries_that_are_no_pages():
    """They do not go back, and nothing is moved from or to them."""
    case, pages = build([30, 30], [3, 5], 4, 30, 5, agree=0.8)
    for r, c, e in ((0, 4, -1), (0, 8, 1 << 30), (1, 1, -7), (1, 2, pages)):
        case["tables"][r][c] = e
    check(case, pages, 4, 30)


@pytest.mark.parametrize("change,status", [
    (dict(nodes=4), 4), (dict(length=3), 8), (dict(length=-1), 8), (dict(offset=-1), 8), (dict(offset=1000), 8),
    (dict(free=range(-40, 0)), 8), (dict(length=1000), 2)])
def test_calls_that_change_nothing(change, status):
    case, pages = build([6, 7, 2], [10, 90, 30], 8, 6)
    if "length" in change:
        case["lengths"][1] = change["length"]
    if "offset" in change:
        case["offsets"][2] = change["offset"]
    nodes = change.get("nodes", 6)
    if "free" in change:  # the stack says that it holds all pages already
        case["free"] = list(range(pages))
        case["drawn"] = [1000] * len(case["drawn"])
        case["tables"] = np.array(case["tables"]).tolist()
        case["lengths"][0], case["offsets"] = case["lengths"][0], case["offsets"]
    want = check(case, pages, 8, nodes)
    assert want["status"] & status


def test_no_drafts_at_all():
    case, pages = build([1, 0, 1], [10, 5, 0], 8, 0)
    case["given"] = [1, 1, 1]
    rows = 3
    want = accept_step(case["lengths"], case["offsets"], case["parents"], case["tokens"], case["drawn"], case["given"],
                       case["tables"], 8, list(case["free"]), pages, 0)
    s = {k: put(v) for k, v in case.items() if k != "free"}
    s.update(free=put(list(case["free"]) + [-5] * (pages - len(case["free"]))), free_count=put([len(case["free"])]),
             lengths_out=put([-9] * rows), free_out=put([-9]), accepted=put(np.full((rows, 1), -9)), accepted_counts=put([-9] * rows),
             last=put([-9] * rows), status=put([-9]), **{"from": None, "to": None})
    paged_accept(s, 8, 0, pages)
    torch.cuda.synchronize()
    for name in ("lengths_out", "accepted", "accepted_counts", "last", "status"):
        assert s[name].reshape(-1).tolist() == np.array(want[name]).reshape(-1).tolist()


@pytest.mark.parametrize("rows", [1023, 1024, 1025, 3000])
def test_many_requests(rows):
    rng = np.random.default_rng(rows)
    case, pages = build(rng.integers(0, 9, rows).tolist(), rng.integers(0, 60, rows).tolist(), 4, 9, rows)
    check(case, pages, 4, 9)


def test_in_place():
    """Lengths and the count of free pages may be written where they were."""
    case, pages = build([8, 9, 3], [10, 3, 0], 2, 9, 2)
    free = list(case["free"])
    want = accept_step(case["lengths"], case["offsets"], case["parents"], case["tokens"], case["drawn"], case["given"],
                       case["tables"], 2, free, pages, 9)
    s = {k: put(v) for k, v in case.items() if k != "free"}
    s.update(free=put(list(case["free"]) + [-5] * (pages - len(case["free"]))), free_count=put([len(case["free"])]),
             accepted=put(np.zeros((3, 10))), accepted_counts=put([0] * 3), last=put([0] * 3), status=put([-9]),
             **{k: put(np.zeros((3, 9))) for k in ("from", "to")})
    s.update(lengths_out=s["lengths"], free_out=s["free_count"])
    paged_accept(s, 2, 9, pages)
    torch.cuda.synchronize()
    assert s["lengths"].tolist() == want["lengths_out"] and s["free_count"].item() == len(free) == want["free_out"]
