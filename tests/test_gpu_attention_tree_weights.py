"""Attention of several new tokens a request holds a softmax's weights in two halves of the type, whatever the number of waves
that share a tile: the tolerance here has no room for weights that are rounded once."""
import pytest
import torch

from paged_common import half_step
from speculate_common import attend_tree64
from test_gpu_attention_tree import Case

pytestmark = pytest.mark.gpu


def outside(case):
    """How far the outputs are beyond what FP32 sums, weights in two halves and the output's rounding allow."""
    out, _ = case.run()
    given = (case.q, case.tables, case.lengths, case.offsets, case.scale, case.positions, case.ancestors, case.window)
    want, _, slack, _ = attend_tree64(case.keys, case.values, *given)
    size = attend_tree64(case.keys, case.values.abs(), *given)[0]  # sum_j p_j |v_j|
    # The slack counts a rounding of each weight to the type, half a step of it.  Of two halves the second is the first's error,
    # which is half a step at most, and is off by half a step of that; the second half of an FP16 weight, which is held
    # times 2^12, may be subnormal: 2^-25 of 2^12 for each key then, of weights whose largest is 1 and whose sum is at least that.
    half = half_step(case.kind)
    slack = slack - size * (half - half * half)
    if case.kind == "fp16":
        slack = slack + 2.0 ** -37 * max(case.lengths) * torch.nan_to_num(case.values.abs()).max().item()
    got = out[:case.offsets[-1]].double().cpu()
    return (got - want).abs() - slack - want.abs() * half - (2.0 ** -25 if case.kind == "fp16" else 0)


# waves that share a tile: one up to 24 rows a request, two up to 72, four from there on
@pytest.mark.parametrize("heads,kv,dim,count", [(4, 1, 64, 4), (4, 1, 64, 12), (4, 1, 64, 30), (16, 1, 128, 1), (16, 1, 128, 3),
                                                (16, 1, 128, 9), (2, 1, 256, 8), (8, 1, 256, 5), (8, 1, 256, 20)])
@pytest.mark.parametrize("chain", [False, True])
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_weights_in_two_halves(kind, chain, heads, kv, dim, count):
    """Scores that differ little, so that the error of theirs is small beside a weight's rounding."""
    case = Case(kind, heads, kv, dim, 16, [9, 14, 0, 40], [count] * 4, chain, seed=count)
    case.scale /= 16
    off = outside(case)
    assert torch.all(off <= 0), (off.max().item(), torch.nonzero(off > 0)[:5].tolist())


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_weights_of_uneven_pages(kind):
    for page, dim in ((7, 64), (20, 128), (3, 256)):
        case = Case(kind, 8, 1, dim, page, [9, 30], [12, 12], False, seed=page)
        case.scale /= 16
        assert torch.all(outside(case) <= 0)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_neighbours_do_not_change_a_request(kind):
    """A request's results are as near whatever the other requests of the call, or its capacity, are."""
    for counts in ([12], [12, 0, 0, 0, 0, 0, 0, 0], [12, 60], [12, 1, 1, 1, 1, 1, 1]):
        case = Case(kind, 4, 1, 128, 16, [20] + [3] * (len(counts) - 1), counts, True, seed=3)
        case.scale /= 16
        assert torch.all(outside(case) <= 0)
