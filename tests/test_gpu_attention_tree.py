"""Attention of several new tokens a request over its pages, against 64 bits: trees and chains, types, head layouts, page
sizes, strides, windows, tokens that see nothing, and what lies where nobody looks."""
import math

import numpy as np
import pytest
import torch

from paged_common import TYPES, describe, half_step, make_cache, make_tables
from speculate_common import attend_tree, attend_tree64, lib, put, random_parents, tree64

pytestmark = pytest.mark.gpu


class Case:
    """Requests of `before` cached and `counts` new tokens; what no token of theirs is in holds NaN."""

    def __init__(self, kind, heads, kv, dim, page, before, counts, chain=False, window=0, layout="token", seed=0, spare=3, words=None):
        rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
        self.kind, self.heads, self.window = kind, heads, window
        self.lengths = [b + c for b, c in zip(before, counts)]
        held = sum(-(-n // page) for n in self.lengths)
        pages = held + spare
        width = max(1, max(-(-n // page) for n in self.lengths)) + 1
        self.tables = make_tables(rng, self.lengths, page, pages, width)
        self.keys, self.values = make_cache(kind, pages, page, kv, dim, layout)
        for r, n in enumerate(self.lengths):
            if n:
                p = torch.tensor([int(self.tables[r][j // page]) for j in range(n)]), torch.tensor([j % page for j in range(n)])
                for c in (self.keys, self.values):
                    c[p[0].cuda(), p[1].cuda()] = torch.randn(n, kv, dim, generator=g).to(TYPES[kind]).cuda()
        self.offsets = np.concatenate([[0], np.cumsum(counts)]).tolist()
        self.tokens = self.offsets[-1] + 2  # two of no request's behind
        self.q = torch.randn(self.tokens, heads * dim, generator=g).to(TYPES[kind]).cuda()
        self.positions = self.ancestors = None
        if not chain:
            parents = sum((random_parents(rng, c) for c in counts), []) + [0, 0]
            self.words = words or -(-max(max(counts), 1) // 32)
            self.positions, self.ancestors = tree64(self.lengths, self.offsets, parents, self.tokens, self.words)
        self.scale = 1 / math.sqrt(dim)

    def run(self, workspace=None):
        t = TYPES[self.kind]
        out = torch.full((self.tokens, self.q.shape[1] + 8), 7.0, dtype=t, device="cuda")[:, :self.q.shape[1]]
        lse = torch.full((self.tokens, self.heads), 7.0, device="cuda")
        tree = {} if self.ancestors is None else {"positions": put(self.positions), "ancestors": put(self.ancestors)}
        attend_tree(describe(self.keys, self.values, self.kind), self.q, self.heads, put(self.tables), put(self.lengths),
                    put(self.offsets), out, lse, scale=self.scale, window=self.window, workspace=workspace, **tree)
        torch.cuda.synchronize()
        return out, lse

    def check(self):
        out, lse = self.run()
        want, e, slack, e_slack = attend_tree64(self.keys, self.values, self.q, self.tables, self.lengths, self.offsets, self.scale,
                                                self.positions, self.ancestors, self.window)
        total = self.offsets[-1]
        got = out[:total].double().cpu()
        off = (got - want).abs() - slack - want.abs() * half_step(self.kind) - (2.0 ** -25 if self.kind == "fp16" else 0)
        assert torch.all(off <= 0), (off.max().item(), torch.nonzero(off > 0)[:5].tolist())
        got = lse[:total].double().cpu()
        assert torch.equal(got == -math.inf, e == -math.inf)
        some = e > -math.inf
        assert torch.all((got - e)[some].abs() <= e_slack[some]), (got - e)[some].abs().max()
        assert torch.all(out[total:] == 7) and torch.all(lse[total:] == 7)  # as they were
        return out, lse


LAYOUTS = [(16, 1, 128), (8, 2, 64), (6, 2, 256), (7, 1, 64), (4, 4, 128), (40, 2, 128), (3, 1, 256)]


@pytest.mark.parametrize("chain", [False, True])
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv,dim", LAYOUTS)
def test_layouts(heads, kv, dim, kind, chain):
    Case(kind, heads, kv, dim, 16, [0, 37, 130, 300, 5], [3, 8, 1, 5, 0], chain).check()


@pytest.mark.parametrize("page", [1, 3, 8, 16, 20, 48, 64, 256])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_pages(page, dim):
    Case("bf16", 8, 1, dim, page, [150, 0, 63, 64], [5, 9, 2, 16], False).check()
    Case("fp16", 4, 2, dim, page, [150, 1, 65], [5, 40, 70], True, window=33).check()


@pytest.mark.parametrize("layout", ["head", "joined", "padded"])
def test_strides(layout):
    Case("bf16", 8, 2, 128, 24, [100, 7], [6, 11], False, layout=layout).check()
    Case("fp16", 8, 2, 64, 16, [100, 7], [6, 11], True, layout=layout).check()


@pytest.mark.parametrize("count", [2, 20, 40])
def test_slots_far_apart(count):
    """Pages side by side and a page's slots 2^24 elements apart, the most that a cache may have."""
    case = Case("bf16", 4, 1, 128, 16, [50, 3], [count, count], False)
    far = []
    for c in (case.keys, case.values):
        room = torch.empty(15 * (1 << 24) + c.shape[0] * 128, dtype=c.dtype, device="cuda")
        far.append(room.as_strided(c.shape, (128, 1 << 24, 128, 1)))
        far[-1].copy_(c)
    case.keys, case.values = far
    case.check()


@pytest.mark.parametrize("heads,kv,dim", [(16, 1, 128), (4, 1, 64), (8, 8, 64), (2, 1, 256)])
@pytest.mark.parametrize("count", [1, 2, 4, 8, 17, 33, 64])
def test_numbers_of_nodes(count, heads, kv, dim):
    """Each number of waves that share a tile, tiles that end anywhere."""
    Case("bf16", heads, kv, dim, 16, [90, 200], [count, count], False, seed=count).check()


@pytest.mark.parametrize("before", [0, 1, 29, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257])
def test_borders_of_tiles(before):
    Case("bf16", 16, 1, 128, 16, [before], [13], False, seed=before).check()
    Case("bf16", 2, 1, 128, 16, [before], [13], True, seed=before).check()
    Case("fp16", 16, 2, 64, 16, [before] * 3, [4] * 3, False, seed=before).check()


@pytest.mark.parametrize("window", [1, 2, 7, 64, 100])
@pytest.mark.parametrize("chain", [False, True])
def test_windows(window, chain):
    Case("bf16", 16, 1, 128, 16, [0, 5, 63, 150, 400], [3, 12, 6, 8, 30], chain, window=window).check()


@pytest.mark.parametrize("count", [33, 100, 300])
def test_long_chains(count):
    """More than one word of nodes, as a tree that is a chain with some branches and as a chain."""
    Case("bf16", 4, 1, 64, 16, [70, 0], [count, 3], False, seed=count).check()
    Case("bf16", 4, 1, 64, 16, [70, 0], [count, 3], True, seed=count).check()


def test_nodes_past_the_words_are_not_seen():
    case = Case("bf16", 4, 1, 64, 16, [40], [50], False, words=2)
    case.ancestors = case.ancestors[:, :1].copy()
    case.check()


def test_many_parts():
    """Few tiles over many keys: parts joined."""
    Case("bf16", 8, 1, 64, 64, [5000], [3], False).check()
    Case("fp16", 16, 2, 128, 64, [3000, 10, 800], [2, 9, 0], True, window=2500).check()
    Case("bf16", 2, 1, 256, 32, [2500, 40], [5, 1], False).check()


def test_many_requests():
    """More than the workgroups look through for themselves, and more than a wave does."""
    rng = np.random.default_rng(4)
    for rows in (65, 300, 1100):
        Case("bf16", 2, 1, 64, 16, rng.integers(0, 40, rows).tolist(), rng.integers(0, 4, rows).tolist(), False, seed=rows).check()
    Case("bf16", 2, 1, 64, 64, [9000 if r == 700 else 3 for r in range(1030)], [2] * 1030, True).check()
    Case("bf16", 2, 1, 64, 64, [9000 if r == 70 else 3 for r in range(80)], [2] * 80, True).check()


@pytest.mark.parametrize("scale", [0.0, -0.09, 2.0])
def test_scales(scale):
    case = Case("bf16", 16, 1, 128, 16, [100, 3], [7, 20], False)
    case.scale = scale
    case.check()


def test_tokens_that_see_nothing():
    case = Case("bf16", 4, 1, 128, 16, [0, 50, 20], [4, 6, 3], False)
    case.ancestors[1] = 0           # no cached tokens before it, and no bit
    case.positions[6] = -1          # a token of no position
    case.tables[2][:] = -1          # pages given back
    out, lse = case.check()
    assert torch.all(lse[[1, 6, 10, 11, 12]] == -math.inf) and torch.all(out[[1, 6, 10, 11, 12]] == 0)


def test_entries_that_are_no_pages():
    case = Case("bf16", 4, 1, 128, 16, [100, 90], [4, 6], False)
    case.tables[0][2], case.tables[1][0], case.tables[1][3] = -1, 1 << 30, case.keys.shape[0]
    case.check()
    case = Case("fp16", 4, 1, 64, 12, [100, 90], [4, 6], True)
    case.tables[0][2], case.tables[1][0], case.tables[1][3] = -1, 1 << 30, case.keys.shape[0]
    case.check()


def test_lengths_that_do_not_hold_the_nodes():
    """Zeros for their tokens, keys past the table not seen, requests of invalid offsets none."""
    case = Case("bf16", 4, 1, 128, 16, [100, 90, 30], [4, 6, 2], False)
    case.lengths[0], case.lengths[1] = 3, -5
    case.check()
    case = Case("bf16", 4, 1, 128, 16, [100, 30], [4, 6], True)
    case.tables = case.tables[:, :4].copy()
    case.check()


@pytest.mark.parametrize("window", [0, 7])
@pytest.mark.parametrize("chain", [False, True])
@pytest.mark.parametrize("length", [-(1 << 31), -(1 << 31) + 1, -(1 << 31) + 2, -17, -1, 0, 2])
def test_lengths_far_below_the_number_of_nodes(length, chain, window):
    case = Case("bf16", 8, 2, 64, 16, [40, 20], [3, 3], chain, window=window)
    case.lengths[0] = length
    out, lse = case.run()
    assert torch.all(out[:3] == 0) and torch.all(lse[:3] == -math.inf)
    case.lengths[0] = 43
    want, e = case.run()
    assert torch.equal(out[3:6], want[3:6]) and torch.equal(lse[3:6], e[3:6])


@pytest.mark.parametrize("full", [False, True])
@pytest.mark.parametrize("heads,count", [(2, 3), (8, 3), (16, 9)])
def test_lengths_past_the_tables(heads, count, full):
    """All tokens see all keys of the table's pages; entries of the last column are no pages.  (Where the last page is not full
    they see what lies behind, which is NaN here.)"""
    case = Case("bf16", heads, 1, 64, 16, [80 - count if full else 70], [count], True)
    case.lengths[0] = case.tables.shape[1] * 16 + count
    out, lse = case.run()
    case.lengths[0] = (1 << 31) - 1
    got, e = case.run()
    assert torch.equal(out.view(torch.int16), got.view(torch.int16)) and torch.equal(lse.view(torch.int32), e.view(torch.int32))
    assert torch.isfinite(lse[:count]).all() if full else torch.isnan(lse[:count]).all()


@pytest.mark.parametrize("odd", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kind,dim", [("bf16", 128), ("fp16", 64), ("bf16", 256)])
@pytest.mark.parametrize("chain", [False, True])
def test_values_that_one_branch_sees(odd, kind, dim, chain):
    """A value that is not finite reaches the tokens that see its key, and no others of its tile."""
    case = Case(kind, 4, 1, dim, 16, [50, 20], [9, 7], chain, window=40)
    page = case.keys.shape[1]
    for r, node in ((0, 3), (1, 6)):
        key = case.lengths[r] - (case.offsets[r + 1] - case.offsets[r]) + node
        case.values[int(case.tables[r][key // page]), key % page, :, 5] = odd
    key = 11  # outside the windows of the later tokens
    case.values[int(case.tables[0][0]), key, :, 40] = odd
    out, lse = case.run()
    want, e, slack, _ = attend_tree64(case.keys, case.values, case.q, case.tables, case.lengths, case.offsets, case.scale,
                                      case.positions, case.ancestors, case.window)
    got = out[:case.offsets[-1]].double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)) and not fine.all() and torch.equal(torch.isnan(want), torch.isnan(got))
    assert torch.equal(got[~fine & ~torch.isnan(got)], want[~fine & ~torch.isnan(got)])
    off = (got - want).abs() - torch.nan_to_num(slack) - want.abs() * half_step(kind) - 2.0 ** -25
    assert torch.all(off[fine] <= 0) and torch.isfinite(lse[:case.offsets[-1]]).all()


@pytest.mark.parametrize("odd", [math.nan, math.inf, -math.inf])
def test_keys_that_one_branch_sees(odd):
    """Scores of a key that is not finite reach the tokens that see it alone."""
    case = Case("bf16", 2, 1, 128, 16, [70], [12], False)
    key = 70 + 4
    sees = (case.ancestors[:, 0] >> 4 & 1).astype(bool)[:12]
    clean, _ = case.run()
    case.keys[int(case.tables[0][key // 16]), key % 16, :, 3] = odd
    out, _ = case.run()
    assert sees.any() and not sees.all()
    assert torch.equal(out[:12][~sees], clean[:12][~sees])


def test_results_do_not_depend_on_the_workspace_or_the_call():
    case = Case("bf16", 16, 1, 128, 16, [1000, 40, 333], [8, 3, 24], False)
    first, e = case.run()
    size = 1 << 27
    for fill in (0, 0x7F):
        again, e2 = case.run(torch.full((size,), fill, dtype=torch.uint8, device="cuda"))
        assert torch.equal(first, again) and torch.equal(e, e2)


def test_in_place():
    """out may be q, row for row."""
    case = Case("bf16", 16, 1, 128, 16, [300, 40], [8, 3], False)
    want, _ = case.run()
    q = case.q.clone()
    attend_tree(describe(case.keys, case.values, "bf16"), q, 16, put(case.tables), put(case.lengths), put(case.offsets), q,
                positions=put(case.positions), ancestors=put(case.ancestors))
    torch.cuda.synchronize()
    assert torch.equal(q[:11], want[:11]) and torch.equal(q[11:], case.q[11:])


def test_two_streams():
    """Calls that run side by side, each with its own workspace, on streams that are not the current one."""
    cases = [Case("bf16", 16, 1, 128, 16, [3000, 40, 333], [8, 3, 24], False), Case("fp16", 8, 2, 64, 16, [2000, 700], [60, 9], True)]
    want = [c.run() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    sizes = [lib().plamo_kernel_attention_paged_tree_workspace(len(c.lengths), c.tokens, c.heads, c.keys.shape[2], c.keys.shape[3]) for c in cases]
    rooms = [torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda") for n in sizes]
    given = []
    for c in cases:
        tree = {} if c.ancestors is None else {"positions": put(c.positions), "ancestors": put(c.ancestors)}
        out = torch.full((c.tokens, c.q.shape[1]), 7.0, dtype=TYPES[c.kind], device="cuda")
        given.append((describe(c.keys, c.values, c.kind), c.q, c.heads, put(c.tables), put(c.lengths), put(c.offsets), out,
                      torch.full((c.tokens, c.heads), 7.0, device="cuda"), tree))
    torch.cuda.synchronize()
    for _ in range(20):
        for s, c, g, room in zip(streams, cases, given, rooms):
            with torch.cuda.stream(s):
                attend_tree(*g[:-1], scale=c.scale, window=c.window, workspace=room, **g[-1])
    torch.cuda.synchronize()
    for g, (out, lse) in zip(given, want):
        assert torch.equal(g[6], out) and torch.equal(g[7], lse)


@pytest.mark.parametrize("rows", [4, 1500])
def test_on_a_graph(rows):
    """Lengths, tables and trees that change between replays; eager calls of the same workspace before each."""
    cases = [Case("bf16", 8, 1, 64, 16, [(r * 37 + 900 * s) % 1100 for r in range(rows)], [(r + s) % 4 for r in range(rows)], False, seed=s)
             for s in range(2)]
    width, tokens = max(c.tables.shape[1] for c in cases), cases[0].tokens
    assert cases[1].tokens == tokens
    pages = max(c.keys.shape[0] for c in cases)
    keys, values = make_cache("bf16", pages, 16, 1, 64, "token")
    tables, lengths, offsets = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in ((rows, width), rows, rows + 1))
    positions, ancestors = torch.zeros(tokens, dtype=torch.int32, device="cuda"), torch.zeros(tokens, 1, dtype=torch.int32, device="cuda")
    q, out = (torch.zeros(tokens, 8 * 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    lse = torch.zeros(tokens, 8, device="cuda")
    room = torch.full((lib().plamo_kernel_attention_paged_tree_workspace(rows, tokens, 8, 1, 64),), 0xFF, dtype=torch.uint8, device="cuda")

    def launch():
        attend_tree(describe(keys, values, "bf16"), q, 8, tables, lengths, offsets, out, lse, positions, ancestors, workspace=room)

    def fill(c):
        for to, of in ((keys, c.keys), (values, c.values), (tables[:, :c.tables.shape[1]], put(c.tables)), (lengths, put(c.lengths)),
                       (offsets, put(c.offsets)), (positions, put(c.positions)), (ancestors, put(c.ancestors)), (q, c.q)):
            to[:of.shape[0]].copy_(of)
        out.fill_(7.0)
        lse.fill_(7.0)

    fill(cases[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        launch()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        launch()
    for turn in range(5):
        c = cases[turn % 2]
        fill(c)
        launch()
        torch.cuda.synchronize()
        want, e = out.clone(), lse.clone()
        room.fill_(0xFF)
        out.fill_(7.0)
        lse.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, e)
        alone, e = c.run()  # (as many tokens: the same division of the work)
        assert torch.equal(out, alone) and torch.equal(lse, e)
