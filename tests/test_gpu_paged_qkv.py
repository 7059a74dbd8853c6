"""Projection rows written into paged caches (plamo_kernel_paged_qkv) against a 64-bit implementation."""
import pytest
import torch

from paged_common import TYPES, describe, half_step, make_cache, paged_qkv, qkv64, rope_words

pytestmark = pytest.mark.gpu


def check(kind, source, dim, heads, kv, tokens, page=16, layout="token", norm=True, rope=True, skip=(), in_place=False):
    g = torch.Generator("cuda").manual_seed(dim * 31 + heads + tokens)
    t = TYPES[kind]
    pages = -(-(tokens + 9) // page) + 1
    keys, values = make_cache(kind, pages, page, kv, dim, layout, fill=3.0)
    wide = (heads + 2 * kv) * dim
    qkv = torch.randn(tokens, wide + 16, generator=g, device="cuda").to(TYPES[source])[:, :wide]
    qkv[0] *= 1e-4   # the small addend under the root counts
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].to(torch.int32)
    positions = torch.randint(0, 500, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    for at, what, value in skip:
        (slots if what == "slot" else positions)[at] = value
    gains = (torch.randn(2, dim, generator=g, device="cuda") * 0.2).to(t) if norm else None
    words, cos, sin = rope_words(500, dim // 2) if rope else (None, None, None)
    want, slack = qkv64(qkv, heads, kv, dim, positions, cos, sin, gains)
    q = qkv if in_place else torch.full((tokens + 1, heads * dim + 8), 5.0, dtype=t, device="cuda")
    before = qkv.clone()
    paged_qkv(describe(keys, values, kind), kind, qkv, heads, slots, q, positions, None if gains is None else gains[0],
              None if gains is None else gains[1], None if words is None else words.cuda())
    torch.cuda.synchronize()

    def near(got, at, part):
        w, s = want[at, part], slack[at, part]
        over = (got.double().cpu() - w).abs() - (w.abs() * half_step(kind) + s * (1 + half_step(kind)) + 2.0 ** -25)
        assert float(over.max()) <= 0, (at, part, float(over.max()))

    untouched_keys, untouched_values = torch.ones(pages * page, dtype=torch.bool), torch.ones(pages * page, dtype=torch.bool)
    for i in range(tokens):
        pos, slot = int(positions[i]), int(slots[i])
        live = 0 <= pos < 500 if rope else pos >= 0
        row = q[i, :heads * dim].view(heads, dim)
        if live:
            near(row, i, slice(0, heads))
        else:
            assert torch.all(row == (before[i, :heads * dim].view(heads, dim) if in_place else 5))
        if live and 0 <= slot < pages * page:
            near(keys[slot // page, slot % page], i, slice(heads, heads + kv))
            near(values[slot // page, slot % page], i, slice(heads + kv, None))
            untouched_keys[slot] = untouched_values[slot] = False
    for cache, rest in ((keys, untouched_keys), (values, untouched_values)):
        assert torch.all(cache.reshape(pages * page, kv, dim)[rest.cuda()] == 3)
    if in_place:
        assert torch.equal(q[:, heads * dim:], before[:, heads * dim:])
    else:
        assert torch.all(q[tokens] == 5) and torch.all(q[:, heads * dim:] == 5)


@pytest.mark.parametrize("kind,source", [("bf16", "fp32"), ("bf16", "bf16"), ("fp16", "fp32"), ("fp16", "fp16")])
@pytest.mark.parametrize("dim,heads,kv", [(128, 16, 1), (64, 6, 3), (256, 2, 2)])
def test_types_and_heads(kind, source, dim, heads, kv):
    check(kind, source, dim, heads, kv, 37)


@pytest.mark.parametrize("tokens", [1, 2, 3, 64, 300])
def test_row_counts(tokens):
    check("bf16", "fp32", 128, 16, 1, tokens, page=7)


@pytest.mark.parametrize("layout", ["head", "joined", "padded"])
def test_orders_in_memory(layout):
    check("bf16", "bf16", 64, 4, 2, 50, layout=layout)


@pytest.mark.parametrize("norm,rope", [(False, True), (True, False), (False, False)])
def test_without_norm_or_rotation(norm, rope):
    check("fp16", "fp32", 128, 4, 1, 20, norm=norm, rope=rope)


def test_skipped_rows():
    skip = [(1, "slot", -1), (4, "slot", 10 ** 6), (5, "position", -1), (9, "position", 500), (11, "position", 2 ** 31 - 1),
            (12, "slot", -2 ** 31)]
    check("bf16", "fp32", 128, 16, 1, 16, skip=skip)
    check("bf16", "bf16", 64, 3, 1, 16, skip=skip)


def test_in_place():
    check("bf16", "bf16", 128, 16, 1, 33, in_place=True)
    check("fp16", "fp16", 256, 2, 1, 33, in_place=True, skip=[(3, "position", -1)])


def test_no_rows():
    keys, values = make_cache("bf16", 2, 16, 1, 64, fill=3.0)
    one = torch.zeros(1, 3 * 64, device="cuda")
    q = torch.full((1, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    slots = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged_qkv(describe(keys, values, "bf16"), "bf16", one[:0], 1, slots, q)
    torch.cuda.synchronize()
    assert torch.all(q == 5) and torch.all(keys == 3) and torch.all(values == 3)


def test_slots_past_two_to_the_31_elements():
    page, dim = 64, 256
    pages = (1 << 31) // (page * dim) + 9
    keys, values = (torch.empty(pages, page, 1, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    qkv = torch.randn(3, 3 * dim, device="cuda")
    slots = torch.tensor([pages * page - 1, (pages - 3) * page + 5, 0], dtype=torch.int32, device="cuda")
    q = torch.zeros(3, dim, dtype=torch.bfloat16, device="cuda")
    paged_qkv(describe(keys, values, "bf16"), "bf16", qkv, 1, slots, q)
    for i, slot in enumerate(slots.tolist()):
        assert torch.equal(keys[slot // page, slot % page, 0], qkv[i, dim:2 * dim].to(torch.bfloat16))
        assert torch.equal(values[slot // page, slot % page, 0], qkv[i, 2 * dim:].to(torch.bfloat16))
    del keys, values
    torch.cuda.empty_cache()


def test_replayed_graph_and_another_stream():
    """Replays with other rows, slots and positions between eager calls, on a stream of their own."""
    g = torch.Generator("cuda").manual_seed(3)
    keys, values = make_cache("bf16", 9, 16, 1, 128, fill=3.0)
    cache = describe(keys, values, "bf16")
    qkv = torch.randn(20, 18 * 128, generator=g, device="cuda")
    slots = torch.arange(20, dtype=torch.int32, device="cuda")
    positions = torch.arange(20, dtype=torch.int32, device="cuda")
    q = torch.zeros(20, 2048, dtype=torch.bfloat16, device="cuda")
    gains = torch.randn(2, 128, generator=g, device="cuda").to(torch.bfloat16)
    words = rope_words(500, 64)[0].cuda()
    call = lambda: paged_qkv(cache, "bf16", qkv, 16, slots, q, positions, gains[0], gains[1], words)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        call()
    for _ in range(4):
        qkv.copy_(torch.randn(20, 18 * 128, generator=g, device="cuda"))
        slots.copy_(torch.randperm(144, generator=g, device="cuda")[:20])
        positions.copy_(torch.randint(0, 500, (20,), generator=g, device="cuda"))
        results = []
        for run in (graph.replay, call):
            q.fill_(5), keys.fill_(3), values.fill_(3)
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                run()
            torch.cuda.synchronize()
            results.append((q.clone(), keys.clone(), values.clone()))
        assert all(torch.equal(a, b) for a, b in zip(*results)) and int((results[0][1] != 3).any(-1).sum()) == 20
