"""Block tables and slot maps built on the GPU (plamo_kernel_paged_tables) against a host allocator that
serves one request after the other.  Everything is whole numbers and has to be equal."""
import random

import pytest
import torch

from paged_common import lib, native, stream, tables_step

pytestmark = pytest.mark.gpu


class Pool:
    """The device arrays of a server, lengths and free_count updated in place."""

    def __init__(self, rows, width, page, pages, capacity, seed=0, room=5):
        put = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        order = list(range(pages))
        random.Random(seed).shuffle(order)
        self.rows, self.width, self.page, self.pages, self.capacity = rows, width, page, pages, capacity
        self.host = {"lengths": [0] * rows, "tables": [[-1] * width for _ in range(rows)], "free": order}
        self.lengths, self.counts = put([0] * rows), put([0] * rows)
        self.tables = put([[-1] * width] * rows)
        self.free, self.free_count = put(order), put([pages])
        self.offsets, self.status = put([-7] * (rows + 1)), put([-7])
        self.slots, self.positions = put([-7] * (capacity + room)), put([-7] * (capacity + room))

    def call(self, lengths_out=None, free_out=None):
        at = lambda t: t.data_ptr()  # noqa: E731
        native.call(lib().plamo_kernel_paged_tables, at(self.lengths), at(self.counts), self.rows, at(self.tables),
                    self.width, self.page, at(self.free), at(self.free_count), self.pages,
                    at(self.lengths if lengths_out is None else lengths_out),
                    at(self.free_count if free_out is None else free_out), at(self.offsets),
                    at(self.slots) if self.capacity else 0, at(self.positions) if self.capacity else 0, self.capacity,
                    at(self.status), stream())

    def step(self, counts, call=None):
        self.counts.copy_(torch.tensor(counts, dtype=torch.int32))
        h = self.host
        want = tables_step(h["lengths"], counts, h["tables"], h["free"], self.page, self.pages, self.capacity)
        (call or self.call)()
        torch.cuda.synchronize()
        self.check(*want)
        return want[3]

    def check(self, offsets, slots, positions, status):
        h = self.host
        assert self.status.item() == status
        assert self.lengths.tolist() == h["lengths"]
        assert self.free_count.item() == len(h["free"])
        assert self.free.tolist()[:len(h["free"])] == h["free"]
        assert self.tables.tolist() == h["tables"]
        assert self.offsets.tolist() == offsets
        c = self.capacity
        assert self.slots.tolist()[:c] == slots and self.positions.tolist()[:c] == positions
        assert self.slots.tolist()[c:] == self.positions.tolist()[c:] == [-7] * (len(self.slots) - c)


@pytest.mark.parametrize("rows,page,width,capacity", [(1, 16, 4, 64), (3, 1, 40, 100), (64, 16, 30, 700), (70, 7, 33, 5000),
                                                      (1000, 64, 9, 20000), (1025, 3, 50, 9000), (2500, 16, 20, 30000)])
def test_steps_of_a_server(rows, page, width, capacity):
    """Prompts, decode steps and requests that end, in random order, until well after the pool has been used
    once; steps that do not fit change nothing."""
    rng = random.Random(rows * 7 + page)
    pool = Pool(rows, width, page, max(2, rows * width // 3), capacity)
    seen = set()
    for turn in range(14):
        counts = []
        for n in pool.host["lengths"]:
            left = width * page - n
            kind = rng.random()
            if n and kind < 0.2:
                counts.append(-1)
            elif kind < 0.3:
                counts.append(0)
            elif kind < 0.6 or n:
                counts.append(min(left, 1))
            else:
                counts.append(min(left, rng.randint(1, max(1, 3 * capacity // (2 * rows)))))
        status = pool.step(counts)
        seen.add(status)
        if status:  # too much at once: one token each
            pool.step([min(1, max(0, c)) if c >= 0 else -1 for c in counts])
    assert 0 in seen


def test_a_long_prompt_and_its_end():
    pool = Pool(2, 5000, 8, 6000, 40000)
    assert pool.step([39999, 1]) == 0
    assert pool.step([0, 0]) == 0
    assert pool.step([-1, 9]) == 0
    assert pool.step([17, -1]) == 0
    assert pool.step([-1, 33000]) == 0


def test_refused_steps_change_nothing():
    pool = Pool(4, 3, 4, 8, 30)
    assert pool.step([5, 4, 0, 1]) == 0
    assert pool.step([8, 1, 0, 0]) == 2          # 13 tokens, 12 fit the table
    assert pool.step([7, 8, 12, 1]) == 1         # 9 pages are needed of 8
    assert pool.step([7, 8, 12, 12]) == 7        # 13 tokens in the last row, and 39 in all of 30
    assert pool.step([-1, -2, 0, 0]) == 8
    pool.lengths[1] = pool.host["lengths"][1] = -1
    assert pool.step([1, 1, 1, 1]) == 8
    pool.lengths[1] = pool.host["lengths"][1] = 4
    assert pool.step([-1, -1, 12, -1]) == 0      # what ends makes room in the same step
    pool.lengths[0] = pool.host["lengths"][0] = 2 ** 31 - 1
    assert pool.step([1, 0, 0, 0]) == 2
    pool.lengths[0] = pool.host["lengths"][0] = 0
    pool.free_count.fill_(9)                     # more than there are pages
    counts = pool.counts.clone()
    pool.call()
    assert pool.status.item() == 8 and pool.free_count.item() == 9 and torch.equal(counts, pool.counts)
    pool.free_count.fill_(-1)
    pool.call()
    assert pool.status.item() == 8 and pool.free_count.item() == -1


def test_exactly_all_pages_tokens_and_columns():
    pool = Pool(3, 4, 5, 12, 60)
    assert pool.step([20, 20, 20]) == 0 and pool.host["free"] == []
    assert pool.step([0, 0, 0]) == 0
    assert pool.step([1, -1, 0]) == 2
    assert pool.step([-1, -1, -1]) == 0 and len(pool.host["free"]) == 12


def test_no_capacity():
    pool = Pool(2, 4, 5, 8, 0)
    assert pool.step([0, 0]) == 0
    assert pool.step([0, 1]) == 4


def test_outputs_of_their_own():
    """lengths_out and free_out elsewhere: the inputs stay, and the same call gives the same again."""
    pool = Pool(5, 6, 4, 30, 50)
    assert pool.step([9, 1, 4, 0, 3]) == 0
    lengths, count = pool.lengths.clone(), pool.free_count.clone()
    outs = torch.full((5,), -7, dtype=torch.int32, device="cuda"), torch.full((1,), -7, dtype=torch.int32, device="cuda")
    for _ in range(3):
        pool.counts.copy_(torch.tensor([4, -1, 1, 2, 0], dtype=torch.int32))
        pool.call(*outs)
        torch.cuda.synchronize()
        assert torch.equal(pool.lengths, lengths) and torch.equal(pool.free_count, count)
    assert pool.step([4, -1, 1, 2, 0]) == 0
    assert torch.equal(outs[0], pool.lengths) and torch.equal(outs[1], pool.free_count)


@pytest.mark.parametrize("capacity", [50, 9000])
def test_replayed_graph(capacity):
    pool = Pool(6, 2000, 8, 6000, capacity)
    pool.step([3, 1, 0, 9, 2, 1])
    graph = torch.cuda.CUDAGraph()
    pool.counts.zero_()
    with torch.cuda.graph(graph):
        pool.call()
    torch.cuda.synchronize()
    for counts in ([1] * 6, [5, -1, 8, 1, 0, 20], [-1, 3, 1, 1, -1, 1], [capacity // 2, 0, 0, 0, 0, 1], [1] * 6):
        pool.step(counts, graph.replay)
        pool.step([1] * 6)


def test_pools_on_two_streams():
    """Two servers' steps in flight at once, each in the order of its own stream."""
    pools = [Pool(40, 30, 16, 500, 700, seed=1), Pool(7, 300, 3, 900, 5000, seed=2)]
    streams = [torch.cuda.Stream() for _ in pools]
    wants = []
    torch.cuda.synchronize()
    for turn in range(6):
        for pool, s in zip(pools, streams):
            counts = [(turn + r) % 5 + (40 if turn == r else 0) for r in range(pool.rows)]
            if turn == 3:
                counts[2] = -1
            h = pool.host
            want = tables_step(h["lengths"], counts, h["tables"], h["free"], pool.page, pool.pages, pool.capacity)
            with torch.cuda.stream(s):
                pool.counts.copy_(torch.tensor(counts, dtype=torch.int32))
                pool.call()
            wants.append(want)
    torch.cuda.synchronize()
    for pool, want in zip(pools, wants[-2:]):
        pool.check(*want)
