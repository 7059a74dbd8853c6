"""Attention of several new tokens a request over its pages: offsets and positions of any kind,
scores that are not finite."""
import math

import numpy as np
import pytest
import torch

from paged_common import describe, half_step, lib
from speculate_common import attend_tree, attend_tree64, put
from test_gpu_attention_tree import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("chain", [False, True])
def test_requests_of_offsets_that_are_none(chain):
    """They have no nodes, and the others' results are what they are without them."""
    case = Case("bf16", 16, 1, 128, 16, [300, 40], [4, 5], chain)
    want, e, slack, e_slack = attend_tree64(case.keys, case.values, case.q, case.tables, case.lengths, case.offsets, case.scale,
                                            case.positions, case.ancestors)
    case.tables, case.lengths = case.tables[[0, 0, 1, 1]], [case.lengths[i] for i in (0, 0, 1, 1)]
    case.offsets = [0, 4, 2 ** 31 - 1, 4, 9]
    out, lse = case.run()
    off = (out[:9].double().cpu() - want).abs() - slack - want.abs() * half_step("bf16")
    assert torch.all(off <= 0) and torch.all((lse[:9].double().cpu() - e).abs() <= e_slack)
    assert torch.all(out[9:] == 7) and torch.all(lse[9:] == 7)
    case.offsets = [-2 ** 31, 4, -1, 4, 9]
    out, lse = case.run()
    off = (out[4:9].double().cpu() - want[4:]).abs() - slack[4:] - want[4:].abs() * half_step("bf16")
    assert torch.all(off <= 0) and torch.all(out[:4] == 7) and torch.all(lse[:4] == 7)


@pytest.mark.parametrize("long_row", [2, 62])
@pytest.mark.parametrize("rows,tokens,heads,kv,dim", [(64, 1000, 16, 1, 128), (300, 90, 8, 2, 64), (1100, 40, 16, 1, 64),
                                                      (64, 500, 4, 1, 256)])
def test_requests_that_overlap(rows, tokens, heads, kv, dim, long_row):
    """Every second request has all tokens, one of them keys of many parts: nothing outside the outputs and the workspace is
    written, and the next call is as if this one had not been."""
    rng, guard = np.random.default_rng(rows), 64
    page, width, pages = 16, 4000, 40
    keys, values = (torch.randn(pages, page, kv, dim, device="cuda").to(torch.bfloat16) for _ in range(2))
    tables = rng.integers(0, pages, (rows, width))
    lengths = np.full(rows, tokens + 50)
    lengths[long_row] = width * page
    size = lib().plamo_kernel_attention_paged_tree_workspace(rows, tokens, heads, kv, dim)
    q = torch.randn(tokens, heads * dim, device="cuda").to(torch.bfloat16)

    def call(offsets, fill):
        room = torch.full((size + 4096,), fill, dtype=torch.uint8, device="cuda")
        out = torch.full((tokens + 2 * guard, heads * dim), 7.0, dtype=torch.bfloat16, device="cuda")
        lse = torch.full((tokens + 2 * guard, heads), 7.0, device="cuda")
        attend_tree(describe(keys, values, "bf16"), q, heads, put(tables), put(lengths), put(offsets), out[guard:-guard], lse[guard:-guard],
                    workspace=room)
        torch.cuda.synchronize()
        for t in (out, lse):
            assert torch.all(t[:guard] == 7) and torch.all(t[-guard:] == 7)
        assert torch.all(room[size:] == fill)
        return out, lse

    ascending = np.minimum(np.arange(rows + 1), tokens)
    want = call(ascending, 0xFF)
    for fill in (0xFF, 0):
        call([0 if r % 2 == 0 else tokens for r in range(rows + 1)], fill)
        call([0 if r % 2 == 0 else tokens - r % 7 for r in range(rows + 1)], fill)
        call(rng.permutation(rows + 1) % (tokens + 1), fill)
        call(rng.integers(-3, tokens + 4, rows + 1), fill)
    assert all(torch.equal(a, b) for a, b in zip(call(ascending, 0), want))


# heads on one KV head and new tokens: 1, 2 and 4 waves a tile, one set of waves or several
SHAPES = [(1, 64, 3), (8, 64, 5), (16, 64, 20), (16, 128, 1), (4, 128, 12), (16, 128, 9), (4, 256, 2), (8, 256, 6), (16, 256, 8)]


@pytest.mark.parametrize("before", [0, 24, 32, 56, 96, 160, 3000])
@pytest.mark.parametrize("heads,dim,count", SHAPES)
def test_nan_alone(heads, dim, count, before):
    """The last key holds NaN, the only key of its tile that is seen or not: the token that sees it has NaN in out and lse, the
    ones before it numbers."""
    case = Case("bf16", heads, 1, dim, 16, [before], [count], True)
    clean, e = case.run()
    at = case.lengths[0] - 1
    case.keys[int(case.tables[0][at // 16]), at % 16, :, 1] = math.nan
    out, lse = case.run()
    assert torch.isnan(out[count - 1]).all() and torch.isnan(lse[count - 1]).all()
    assert torch.equal(out[:count - 1], clean[:count - 1]) and torch.equal(lse[:count - 1], e[:count - 1])


@pytest.mark.parametrize("before", [0, 5, 40, 200, 3000])
@pytest.mark.parametrize("heads,dim,count", SHAPES)
def test_a_row_of_nan(heads, dim, count, before):
    """All scores of one query row are NaN, and no other row's."""
    case = Case("fp16", heads, 1, dim, 16, [before], [count], False)
    clean, e = case.run()
    token, head = count // 2, heads - 1
    case.q[token, head * dim + 7] = math.nan
    out, lse = case.run()
    rows, want = out[:count].view(count, heads, dim), clean[:count].view(count, heads, dim)
    assert torch.isnan(rows[token, head]).all() and torch.isnan(lse[token, head])
    others = torch.ones(count, heads, dtype=torch.bool, device="cuda")
    others[token, head] = False
    assert torch.equal(rows[others], want[others]) and torch.equal(lse[:count][others], e[:count][others])


@pytest.mark.parametrize("before", [0, 40, 200])
@pytest.mark.parametrize("heads,dim,count", SHAPES)
def test_scores_of_minus_infinity(heads, dim, count, before):
    """A row of such scores alone gives zeros and minus infinity, beside one whose scores are numbers."""
    case = Case("bf16", heads, 1, dim, 16, [before, 30], [count, 2], True)
    for j in range(case.lengths[0]):
        case.keys[int(case.tables[0][j // 16]), j % 16] = 0
        case.keys[int(case.tables[0][j // 16]), j % 16, :, 0] = -math.inf
    case.q.view(-1, heads, dim)[:, :, 0] = 1
    out, lse = case.run()
    assert torch.all(out[:count] == 0) and torch.all(lse[:count] == -math.inf)
    assert torch.isfinite(out[count:count + 2]).all() and torch.isfinite(lse[count:count + 2]).all()


@pytest.mark.parametrize("window", [1, 20, 64, 2 ** 31 - 1])
@pytest.mark.parametrize("heads,dim,count", SHAPES[::2])
def test_positions_before_the_nodes(heads, dim, count, window):
    """They count as the first node's, which sees the window's last keys before it; any position behind is its own."""
    case = Case("bf16", heads, 1, dim, 16, [100, 70], [count, count], False, window=window)
    first = [100] * count + [70] * count
    case.positions[:2 * count] = first
    want = case.run()
    case.positions[:2 * count] = [(0, 1, p - 1, p // 2)[i % 4] for i, p in enumerate(first)]
    assert all(torch.equal(a, b) for a, b in zip(case.run(), want))
    case.positions[:2 * count] = [(p + 5, 2 ** 31 - 1)[i % 2] for i, p in enumerate(first)]
    case.check()


@pytest.mark.parametrize("kv,heads,dim", [(256, 256, 64), (100, 200, 128), (256, 512, 64)])
def test_many_kv_heads(kv, heads, dim):
    """Fewer parts aimed at than there are tiles, down to one."""
    Case("bf16", heads, kv, dim, 16, [400, 3], [2, 1], False).check()
    Case("fp16", heads, kv, dim, 16, [300], [3], True, window=200).check()


def test_most_requests():
    """2^20 requests of one token, which sees its own key alone: its value, bit for bit."""
    rows, dim = 1 << 20, 64
    keys, values, q = (torch.randn(rows, dim, device="cuda").to(torch.bfloat16) for _ in range(3))
    tables = torch.randperm(rows, device="cuda").int().view(rows, 1)
    lengths, offsets = torch.ones(rows, dtype=torch.int32, device="cuda"), torch.arange(rows + 1, dtype=torch.int32, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros(rows, 1, device="cuda")
    attend_tree(describe(keys.view(rows, 1, 1, dim), values.view(rows, 1, 1, dim), "bf16"), q, 1, tables, lengths, offsets, out, lse)
    torch.cuda.synchronize()
    page = tables[:, 0].long()
    assert torch.equal(out, values[page])
    score = (q.double() * keys[page].double()).sum(1) / 8
    size = (q.double() * keys[page].double()).abs().sum(1) / 8
    # (as in attend_tree64: sums of `dim` products, then the logarithm)
    assert torch.all((lse[:, 0].double() - score).abs() <= size * (dim + 4) * 2.0 ** -23 + 2.0 ** -20 + score.abs() * 2.0 ** -21)


@pytest.mark.parametrize("heads,dim", [(1, 64), (2, 128), (1, 256)])
@pytest.mark.parametrize("before", [0, 1000])
def test_long_chains_of_a_window_of_one(heads, dim, before):
    """Tiles that see few of their request's keys, parts that hold none."""
    count, page = 30000, 64
    pages = -(-(before + count) // page)
    keys, values = (torch.randn(pages, page, 1, dim, device="cuda").to(torch.bfloat16) for _ in range(2))
    tables = torch.randperm(pages, device="cuda").int().view(1, pages)
    q = torch.randn(count, heads * dim, device="cuda").to(torch.bfloat16)
    out = torch.zeros_like(q)
    attend_tree(describe(keys, values, "bf16"), q, heads, tables, put([before + count]), put([0, count]), out, window=1)
    torch.cuda.synchronize()
    own = values[tables[0].long(), :, 0].reshape(-1, dim)[before:before + count]
    assert torch.equal(out.view(count, heads, dim), own[:, None].expand(count, heads, dim))
