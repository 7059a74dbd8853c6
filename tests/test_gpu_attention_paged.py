"""Attention over paged caches (plamo_kernel_attention_paged) against a 64-bit implementation.

What the cache holds outside the tokens of a request is NaN in every test, table entries behind its
pages are -1, and the workspace starts out as 0xff bytes: none of them may reach an output."""
import math

import numpy as np
import pytest
import torch

from paged_common import TYPES, attend, attend64, describe, half_step, make_cache, make_tables

pytestmark = pytest.mark.gpu


def build(kind, dim, heads, kv, page, lengths, layout="token", seed=0, spare=3, width=None, window=0):
    rng = np.random.default_rng([seed, dim, heads, page, len(lengths)])
    held = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(held) + spare
    width = width or max(1, max(held))
    tables = make_tables(rng, [max(n, 0) for n in lengths], page, pages, width)
    keys, values = make_cache(kind, pages, page, kv, dim, layout)
    for r, n in enumerate(lengths):
        for c in range(-(-max(n, 0) // page)):
            live = min(page, n - c * page)
            for cache in (keys, values):
                new = torch.from_numpy(rng.standard_normal((live, kv, dim))).to(TYPES[kind]).cuda()
                cache[int(tables[r, c]), :live] = new
            if window and (c + 1) * page <= n - window:  # behind the window: given back, its entry gone
                keys[int(tables[r, c])] = values[int(tables[r, c])] = float("nan")
                tables[r, c] = -1
    q = torch.full((len(lengths), heads * dim + 8), float("nan"), dtype=TYPES[kind], device="cuda")[:, :heads * dim]
    q.copy_(torch.from_numpy(rng.standard_normal((len(lengths), heads * dim))))
    return keys, values, tables, q


def check(kind, keys, values, tables, q, lengths, window=0, scale=None, workspace=None):
    rows, wide = q.shape
    dim, heads = keys.shape[3], wide // keys.shape[3]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out = torch.full((rows + 1, wide + 16), 7.0, dtype=TYPES[kind], device="cuda")
    lse = torch.full((rows + 1, heads), 7.0, device="cuda")
    attend(describe(keys, values, kind), q, heads, torch.from_numpy(tables).cuda(),
           torch.tensor(lengths, dtype=torch.int32, device="cuda"), out, lse, scale, window, workspace)
    torch.cuda.synchronize()
    assert torch.all(out[rows] == 7) and torch.all(out[:, wide:] == 7) and torch.all(lse[rows] == 7)
    want, norm, slack, norm_slack = attend64(keys, values, q, tables, lengths, scale, window)
    got = out[:rows, :wide].double().cpu()
    over = (got - want).abs() - (want.abs() * half_step(kind) + slack * (1 + half_step(kind)) + 1e-7)
    assert torch.isfinite(got).all() and float(over.max()) <= 0, float(over.max())
    seen = torch.isfinite(norm)
    log = lse[:rows].double().cpu()
    assert torch.equal(torch.isfinite(log), seen) and torch.all(log[~seen] == -math.inf)
    assert torch.all((log - norm).abs()[seen] <= norm_slack[seen])
    assert torch.all(got.view(rows, heads, dim)[~seen] == 0)
    return out[:rows, :wide].clone(), lse[:rows].clone()


LENGTHS = [1, 0, 15, 16, 17, 31, 32, 33, 127, 128, 129, 500]


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,heads,kv", [(128, 16, 1), (64, 6, 2), (256, 4, 4), (128, 40, 2), (64, 7, 1), (256, 17, 1)])
@pytest.mark.parametrize("page", [16, 5])
def test_heads_types_and_pages(kind, dim, heads, kv, page):
    check(kind, *build(kind, dim, heads, kv, page, LENGTHS), LENGTHS)


@pytest.mark.parametrize("page", [1, 8, 24, 48, 64, 100, 256])
def test_page_sizes(page):
    lengths = [700, 1, 257, 64, 0]
    check("bf16", *build("bf16", 128, 8, 2, page, lengths), lengths)


@pytest.mark.parametrize("layout", ["head", "joined", "padded"])
@pytest.mark.parametrize("page", [16, 20])
def test_orders_in_memory(layout, page):
    lengths = [333, 2, 90]
    check("fp16", *build("fp16", 64, 8, 4, page, lengths, layout), lengths)


@pytest.mark.parametrize("window", [1, 16, 100, 2048])
@pytest.mark.parametrize("page", [16, 12])
def test_window(window, page):
    lengths = [1, 99, 100, 101, 117, 2047, 2048, 2049, 3001, 0]
    check("bf16", *build("bf16", 128, 4, 1, page, lengths, window=window), lengths, window)


def test_one_long_row_and_many_short():
    lengths = [20011] + [3] * 70 + [1500, 0, 777]
    check("bf16", *build("bf16", 128, 16, 1, 64, lengths), lengths)


def test_rows_past_a_wave_and_one_row():
    lengths = [(37 * r) % 211 for r in range(300)]
    check("fp16", *build("fp16", 64, 2, 1, 16, lengths), lengths)
    check("fp16", *build("fp16", 64, 2, 1, 16, [5001]), [5001])


def test_pages_that_are_none_are_not_seen():
    lengths = [400, 300, 40]
    keys, values, tables, q = build("bf16", 128, 16, 1, 16, lengths)
    tables[0, 3] = -5
    tables[0, 7] = keys.shape[0]
    tables[1, 0] = 2 ** 31 - 1
    tables[2, :] = -1          # nothing left of the row
    check("bf16", keys, values, tables, q, lengths)
    keys, values, tables, q = build("bf16", 128, 16, 1, 10, lengths)
    tables[0, 3], tables[1, 29], tables[2, :] = -5, keys.shape[0], 2 ** 31 - 1
    check("bf16", keys, values, tables, q, lengths)


def test_lengths_below_zero_and_past_the_table():
    lengths = [48, 48, 30]
    keys, values, tables, q = build("bf16", 64, 4, 1, 16, lengths)
    check("bf16", keys, values, tables, q, [-3, 2 ** 31 - 1, 30])


def test_shared_pages():
    lengths = [200, 200, 170]
    keys, values, tables, q = build("bf16", 128, 16, 1, 16, lengths)
    tables[1, :9] = tables[0, :9]
    tables[2, :] = tables[0, :]
    check("bf16", keys, values, tables, q, lengths)


def test_scales():
    lengths = [300, 17]
    data = build("bf16", 128, 16, 1, 16, lengths)
    for scale in (0.0, -0.1, 1.0):
        check("bf16", *data, lengths, scale=scale)


def test_weights_that_differ_by_orders():
    """One key far above thousands of others, which count together; FP16's range of weights."""
    for kind in ("bf16", "fp16"):
        n = 6000
        keys, values, tables, q = build(kind, 64, 1, 1, 16, [n])
        keys.mul_(0.02)
        keys[int(tables[0, 2]), 3, 0] = q[0] / q[0].float().norm() * 8
        check(kind, keys, values, tables, q, [n], scale=1.0)


def test_scores_of_minus_infinity_weigh_nothing():
    keys, values, tables, q = build("bf16", 64, 2, 1, 16, [100, 40])
    q.abs_()
    low = keys[int(tables[0, 1]), 0:5]
    low.fill_(-math.inf)
    for c in range(3):
        keys[int(tables[1, c])] = -math.inf
    out = torch.zeros(2, 128, dtype=torch.bfloat16, device="cuda")
    lse = torch.zeros(2, 2, device="cuda")
    attend(describe(keys, values, "bf16"), q, 2, torch.from_numpy(tables).cuda(),
           torch.tensor([100, 40], dtype=torch.int32, device="cuda"), out, lse)
    seen = [j for j in range(100) if not 16 <= j < 21]
    at = torch.tensor([int(tables[0, j // 16]) for j in seen]).cuda(), torch.tensor([j % 16 for j in seen]).cuda()
    k, v = keys[at][:, 0].double(), values[at][:, 0].double()
    share = torch.softmax(q[0].double().view(2, 64) @ k.T / 8, -1)
    assert torch.all((out[0].double().view(2, 64) - share @ v).abs() <= (share @ v).abs() * 2.0 ** -8 + 2.0 ** -12)
    assert torch.all(out[1] == 0) and torch.all(lse[1] == -math.inf)


def test_the_same_call_gives_the_same_bits():
    lengths = [5000, 40, 1300, 0]
    data = build("bf16", 128, 16, 1, 64, lengths)
    first = check("bf16", *data, lengths)
    for _ in range(3):
        again = check("bf16", *data, lengths)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_elements_past_two_to_the_31():
    page, kv, dim = 16, 8, 128
    pages = (1 << 31) // (page * kv * dim) + 5
    keys, values = (torch.empty(pages, page, kv, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for chosen in ([pages - 1, 0, pages - 2, 3], [pages - 3, pages - 4, pages - 1, pages - 2]):
        tables = np.array([chosen], np.int32)
        for c in chosen:
            keys[c], values[c] = (torch.randn(page, kv, dim, device="cuda") for _ in range(2))
        q = torch.randn(1, 8 * dim, device="cuda").to(torch.bfloat16)
        check("bf16", keys, values, tables, q, [61])
    del keys, values
    torch.cuda.empty_cache()


def test_another_stream():
    lengths = [900, 33]
    keys, values, tables, q = build("bf16", 128, 16, 1, 16, lengths)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        check("bf16", keys, values, tables, q, lengths)


def test_two_graphs_with_their_own_workspaces():
    """Replayed several times with other lengths, between eager calls, and one after the other on two streams."""
    cases = []
    for seed, lengths in ((1, [2500, 70, 900]), (2, [130, 4000])):
        keys, values, tables, q = build("bf16", 128, 16, 1, 16, lengths, seed=seed)
        device = torch.from_numpy(tables).cuda()
        size = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        out = torch.zeros(len(lengths), 2048, dtype=torch.bfloat16, device="cuda")
        cache = describe(keys, values, "bf16")
        work = attend(cache, q, 16, device, size, out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attend(cache, q, 16, device, size, out, workspace=work)
        cases.append((graph, keys, values, tables, q, device, size, out, work, torch.cuda.Stream()))
    for turn in range(4):
        for graph, *_, size, out, _, s in cases:
            out.fill_(7)
            size.copy_(torch.tensor([max(1, n - 117 * turn) for n in size.tolist()], dtype=torch.int32))
        torch.cuda.synchronize()
        for graph, *_, s in cases:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for graph, keys, values, tables, q, _, size, out, _, _ in cases:
            eager, _ = check("bf16", keys, values, tables, q, size.tolist())
            assert torch.equal(eager, out)


@pytest.mark.parametrize("page", [16, 20])
def test_many_rows_in_parts(page):
    """Enough rows that several heads' parts are joined at once, and heads that this does not divide."""
    lengths = [(389 * r) % 1501 for r in range(240)]
    check("bf16", *build("bf16", 64, 18, 3, page, lengths), lengths)


@pytest.mark.parametrize("rows,kv,most", [(3, 1, 239), (3, 1, 241), (90, 3, 490), (90, 3, 500), (80, 3, 500)])
@pytest.mark.parametrize("page", [1, 16])
def test_rows_in_one_part(rows, kv, most, page):
    """Beside the widths up to which a row is not divided."""
    lengths = [most - (61 * r) % most for r in range(rows)]
    check("fp16", *build("fp16", 64, 2 * kv, kv, page, lengths), lengths)


@pytest.mark.parametrize("window", [239, 241, 242, 497])
def test_windows_in_one_part(window):
    lengths = [4000 - 133 * r for r in range(30)]
    for kv in (1, 9):
        check("bf16", *build("bf16", 64, kv, kv, 16, lengths, window=window), lengths, window)


def test_nan_and_infinite_scores_are_the_formulas():
    """NaN in a visible key, or a score of infinity, makes the rows and heads that see it NaN, no others."""
    lengths = [700, 640, 700]
    for page in (16, 10):
        keys, values, tables, q = build("bf16", 64, 4, 2, page, lengths)
        q.abs_()
        plain = torch.zeros(3, 256, dtype=torch.bfloat16, device="cuda")
        out = plain.clone()
        args = describe(keys, values, "bf16"), q, 4, torch.from_numpy(tables).cuda()
        size = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        attend(*args, size, plain)
        keys[int(tables[0, 320 // page]), 0, 1, 5] = math.nan
        keys[int(tables[2, 320 // page]), 0, 0, 5] = math.inf
        attend(*args, size, out)
        out, plain = out.view(3, 2, 2, 64), plain.view(3, 2, 2, 64)
        assert torch.isnan(out[0, 1]).all() and torch.isnan(out[2, 0]).all()
        assert torch.equal(out[1], plain[1]) and torch.equal(out[0, 0], plain[0, 0]) and torch.equal(out[2, 1], plain[2, 1])


@pytest.mark.parametrize("lengths", [[5000, 3, 0, 1300], [90, 200, 1]])
def test_output_in_place_of_the_queries(lengths):
    keys, values, tables, q = build("bf16", 128, 16, 1, 16, lengths)
    want, _ = check("bf16", keys, values, tables, q, lengths)
    attend(describe(keys, values, "bf16"), q, 16, torch.from_numpy(tables).cuda(),
           torch.tensor(lengths, dtype=torch.int32, device="cuda"), q)
    assert torch.equal(q, want)


@pytest.mark.parametrize("rows", [1024, 1025, 2100])
def test_more_rows_than_workgroups_search(rows):
    lengths = [(53 * r) % 331 for r in range(rows)]
    lengths[rows // 2], lengths[rows - 1] = 6001, 2000
    check("bf16", *build("bf16", 64, 3, 1, 16, lengths), lengths)
    check("fp16", *build("fp16", 64, 2, 2, 20, lengths[:1030], window=300), lengths[:1030], 300)


def test_very_many_rows():
    """One key each: the output is its value."""
    rows = 70001
    keys, values = make_cache("bf16", rows, 16, 1, 64, fill=float("nan"))
    g = torch.Generator("cuda").manual_seed(5)
    keys[:, 0] = torch.randn(rows, 1, 64, generator=g, device="cuda").to(torch.bfloat16)
    values[:, 0] = torch.randn(rows, 1, 64, generator=g, device="cuda").to(torch.bfloat16)
    pages = torch.randperm(rows, generator=g, device="cuda").to(torch.int32)
    q = torch.randn(rows, 128, generator=g, device="cuda").to(torch.bfloat16)
    size = torch.ones(rows, dtype=torch.int32, device="cuda")
    for width in (1, 20):
        tables = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
        tables[:, 0] = pages
        out = torch.zeros(rows, 128, dtype=torch.bfloat16, device="cuda")
        attend(describe(keys, values, "bf16"), q, 2, tables, size, out)
        want = values[pages.long(), 0]
        assert torch.equal(out.view(rows, 2, 64), want.expand(rows, 2, 64))


@pytest.mark.parametrize("rows,most", [(1, 90), (7, 200), (9, 700), (30, 1500), (1030, 300)])
@pytest.mark.parametrize("page", [16, 9])
def test_several_tiles_of_heads(rows, most, page):
    """33 heads on one KV head are three tiles of a part: alone, in parts, and of listed parts."""
    lengths = [most - (29 * r) % most for r in range(rows)]
    check("bf16", *build("bf16", 64, 33, 1, page, lengths), lengths)
    if rows < 100:
        check("fp16", *build("fp16", 128, 36, 2, page, lengths), lengths)
