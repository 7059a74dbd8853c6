"""Table entries and free pages that are no pages (plamo_kernel_paged_tables): behind a sliding window a request's
pages have been given back and their entries are -1, and a caller's mistake can leave anything on the stack.  Only
pages 0 .. pages - 1 go back, and a step that would place tokens in anything else changes nothing.  Whole numbers,
which have to be equal to those of a host allocator."""
import random

import pytest
import torch

from paged_common import tables_step
from test_gpu_paged_tables import Pool

pytestmark = pytest.mark.gpu

NONE = [-1, -5, 2 ** 31 - 1, -2 ** 31]


def pool_step(lengths, counts, tables, free, page, pages, capacity):
    """tables_step where entries may be no pages: lists changed in place, nothing with a status other than 0."""
    is_page = lambda e: 0 <= e < pages  # noqa: E731
    back = [e for n, c, row in zip(lengths, counts, tables) if c < 0 for e in row[:-(-n // page)] if is_page(e)]
    new = [-(-(n + c) // page) - -(-n // page) for n, c in zip(lengths, counts) if c >= 0]
    stack = free + back
    popped = stack[len(stack) - sum(new):] if sum(new) else []
    partial = [row[n // page] for n, c, row in zip(lengths, counts, tables) if c > 0 and n % page]
    status = 8 if len(stack) > pages else 1 if sum(new) > len(stack) else 0
    if sum(max(c, 0) for c in counts) > capacity:
        status |= 4
    if not status and not all(map(is_page, popped + partial)):
        status = 8
    if status:
        return [0] * (len(lengths) + 1), [-1] * capacity, [-1] * capacity, status
    # requests that end keep nothing: the rest is an ordinary step
    free[:] = stack
    ended = [c < 0 for c in counts]
    for r, e in enumerate(ended):
        if e:
            lengths[r] = 0
    return tables_step(lengths, [0 if e else c for e, c in zip(ended, counts)], tables, free, page, pages, capacity)


class Window(Pool):
    """A pool whose requests' older pages the caller gives back itself."""

    def step(self, counts, call=None):
        h = self.host
        self.counts.copy_(torch.tensor(counts, dtype=torch.int32))
        before = [list(h["lengths"]), [list(r) for r in h["tables"]], list(h["free"]), self.free.tolist()]
        want = pool_step(h["lengths"], counts, h["tables"], h["free"], self.page, self.pages, self.capacity)
        (call or self.call)()
        torch.cuda.synchronize()
        self.check(*want)
        if want[3]:
            assert [h["lengths"], h["tables"], h["free"]] == before[:3] and self.free.tolist() == before[3]
        return want[3]

    def upload(self):
        h = self.host
        self.tables.copy_(torch.tensor(h["tables"], dtype=torch.int32))
        self.free[:len(h["free"])] = torch.tensor(h["free"], dtype=torch.int32)
        self.free_count.fill_(len(h["free"]))

    def drop(self, r, entries, gone=-1):
        """The caller takes pages out of a request's table and puts them on the stack."""
        row = self.host["tables"][r]
        for i in entries:
            if 0 <= row[i] < self.pages:
                self.host["free"].append(row[i])
                row[i] = gone
        self.upload()


def test_a_window_ends_while_another_grows():
    pool = Window(2, 8, 4, 9, 40)
    assert pool.step([30, 4]) == 0
    pool.drop(0, range(5))
    assert pool.step([-1, 28]) == 0
    assert sorted(pool.host["free"] + pool.host["tables"][1]) == list(range(9))
    assert min(pool.slots.tolist()[:28]) >= 0


@pytest.mark.parametrize("gone", NONE)
def test_a_request_whose_pages_are_all_gone(gone):
    pool = Window(3, 6, 4, 13, 40)
    assert pool.step([24, 9, 0]) == 0
    pool.drop(0, range(6), gone)
    assert pool.step([-1, 1, 0]) == 0          # nothing goes back
    assert len(pool.host["free"]) == 10
    pool.drop(1, [0, 2], gone)
    assert pool.step([5, -1, 20]) == 0


@pytest.mark.parametrize("rows,page,width", [(7, 16, 40), (300, 3, 9), (1024, 8, 5), (1025, 4, 12), (2500, 16, 20)])
def test_holes_anywhere(rows, page, width):
    rng = random.Random(rows + page)
    pool = Window(rows, width, page, rows * width // 2, rows * page)
    seen = set()
    for turn in range(10):
        counts = []
        for n in pool.host["lengths"]:
            kind = rng.random()
            counts.append(-1 if n and kind < 0.3 else 0 if kind < 0.4 else
                          min(width * page - n, rng.randint(1, max(1, page))))
        seen.add(pool.step(counts))
        for r, n in enumerate(pool.host["lengths"]):  # all but the page that is being filled
            if rng.random() < 0.5:
                row, whole = pool.host["tables"][r], n // page
                for i in rng.sample(range(whole), rng.randint(0, whole)):
                    if 0 <= row[i] < pool.pages:
                        pool.host["free"].append(row[i])
                        row[i] = rng.choice(NONE + [pool.pages])
        pool.upload()
    assert 0 in seen


def test_a_long_request_with_holes_ends():
    pool = Window(2, 6000, 8, 7000, 50000)
    assert pool.step([47999, 1]) == 0
    pool.drop(0, [i for i in range(5999) if i % 7 == 3 or 900 < i < 2100])
    assert pool.step([-1, 30000]) == 0
    assert pool.step([9, -1]) == 0


@pytest.mark.parametrize("gone", NONE + [9])
def test_free_pages_that_are_none_are_not_given(gone):
    pool = Window(2, 8, 4, 9, 40)
    assert pool.step([4, 0]) == 0
    pool.host["free"][5] = gone                # of eight free ones
    pool.upload()
    assert pool.step([0, 8]) == 0              # two from above it
    assert pool.step([0, 5]) == 8              # the third one, and the one that is none
    assert pool.step([0, 4]) == 8
    assert pool.step([-1, 4]) == 0             # the page that goes back lies above it
    assert pool.step([1, -1]) == 0


def test_far_down_the_stack():
    pool = Window(2, 5000, 4, 6000, 20000)
    pool.host["free"][1500] = -1               # 4,499 lie above it
    pool.upload()
    assert pool.step([4 * 4499, 1]) == 8
    assert pool.step([4 * 4499, 0]) == 0
    assert pool.step([-1, 4 * 4499]) == 0
    assert pool.step([1, 0]) == 8


@pytest.mark.parametrize("gone", NONE + [30])
def test_no_token_goes_into_a_page_that_is_none(gone):
    pool = Window(3, 6, 5, 30, 40)
    assert pool.step([7, 12, 10]) == 0
    pool.host["tables"][1][2] = gone           # two of its five places are taken
    pool.upload()
    assert pool.step([1, 1, 1]) == 8
    assert pool.step([1, 0, 1]) == 0
    assert pool.step([1, -1, 1]) == 0
    pool.host["tables"][2][1] = gone           # full: no new token lies there
    pool.upload()
    assert pool.step([1, 3, 1]) == 0


@pytest.mark.parametrize("capacity", [50, 9000])
def test_replayed_with_holes(capacity):
    pool = Window(4, 1000, 8, 2000, capacity)
    pool.step([30, 41, 0, 9])
    graph = torch.cuda.CUDAGraph()
    pool.counts.zero_()
    with torch.cuda.graph(graph):
        pool.call()
    torch.cuda.synchronize()
    for counts in ([1] * 4, [-1, 20, 3, 1], [5, -1, 1, 0], [1, 1, 1, -1]):
        pool.drop(0, range(pool.host["lengths"][0] // 8))
        pool.drop(1, range(0, pool.host["lengths"][1] // 8, 2))
        assert pool.step(counts, graph.replay) == 0
        assert pool.step([1] * 4) == 0
