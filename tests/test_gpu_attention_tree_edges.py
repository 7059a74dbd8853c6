"""Attention of several new tokens a request over its pages: offsets of any kind."""
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
