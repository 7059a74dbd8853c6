"""Keys and values moved from slot to slot in all layers: whole pools compared, bit for bit."""
import numpy as np
import pytest
import torch

from paged_common import describe, make_cache
from speculate_common import paged_move, put

pytestmark = pytest.mark.gpu


def pools(layers, kind, pages, page, kv, dim, layout, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    made = []
    for _ in range(layers):
        keys, values = make_cache(kind, pages, page, kv, dim, layout)
        for c in (keys, values):
            c.copy_(torch.randn(c.shape, generator=g, device="cuda"))
        made.append((keys, values))
    return made


def moved(cache, source, target):
    """A move after the other of each group."""
    flat = cache.reshape(-1, *cache.shape[2:]).clone()
    slots = flat.shape[0]
    for row_from, row_to in zip(source, target):
        for a, b in zip(row_from, row_to):
            if 0 <= a < slots and 0 <= b < slots:
                flat[b] = flat[a]
    return flat.reshape(cache.shape)


def check(made, kind, source, target):
    want = [[moved(c.cpu(), source, target) for c in pair] for pair in made]
    paged_move([describe(k, v, kind) for k, v in made], put(source), put(target))
    torch.cuda.synchronize()
    for pair, w in zip(made, want):
        for got, x in zip(pair, w):
            assert torch.equal(got.cpu().view(torch.int16), x.view(torch.int16))


def paths(rng, slots, groups, group):
    """Kept nodes of each group's own slots to its first places, as accepted paths are."""
    own = rng.permutation(slots)[:groups * (group + 1)].reshape(groups, group + 1)
    source, target = np.full((groups, group), -1), np.full((groups, group), -1)
    for g in range(groups):
        kept = [i for i in range(1, group + 1) if rng.random() < 0.6]
        for j, k in enumerate(kept):
            if k != j + 1:
                source[g, j], target[g, j] = own[g, k], own[g, j + 1]
    return source.tolist(), target.tolist()


@pytest.mark.parametrize("layout", ["token", "head", "joined", "padded"])
@pytest.mark.parametrize("kind,kv,dim,page", [("bf16", 1, 128, 16), ("fp16", 3, 64, 5), ("bf16", 2, 256, 1), ("fp16", 8, 128, 64)])
def test_accepted_paths(kind, kv, dim, page, layout):
    rng = np.random.default_rng(3)
    pages = -(-200 // page)
    for group in (1, 3, 7, 8, 9, 16, 17):
        check(pools(2, kind, pages, page, kv, dim, layout, group), kind, *paths(rng, pages * page, 200 // (group + 1), group))


@pytest.mark.parametrize("layers", [1, 3, 64, 65, 130])
def test_layers(layers):
    rng = np.random.default_rng(4)
    check(pools(layers, "bf16", 9, 4, 1, 64, "token"), "bf16", *paths(rng, 36, 5, 6))


@pytest.mark.parametrize("count", [1, 2, 63, 64, 65, 1000])
def test_copies(count):
    rng = np.random.default_rng(count)
    slots = rng.permutation(2048)[:2 * count].reshape(2, count, 1) if count <= 1000 else None
    check(pools(2, "bf16", 128, 16, 2, 128, "token", count), "bf16", slots[0].tolist(), slots[1].tolist())


def test_one_source_many_targets():
    check(pools(1, "bf16", 8, 16, 1, 128, "token"), "bf16", [[3]] * 20, [[i] for i in range(20, 40)])


def test_a_long_group_moves_up():
    """One group of more moves than are read ahead, each from the slot of a later one."""
    n = 100
    check(pools(1, "bf16", 8, 16, 1, 128, "token"), "bf16", [list(range(2, n + 2))], [list(range(1, n + 1))])


def test_slots_that_are_none():
    check(pools(1, "fp16", 8, 16, 1, 64, "token"), "fp16", [[-1, 5, 128, 7, 2 ** 31 - 1, 9]], [[3, -1, 4, 128, 6, 60]])


def test_nothing_to_move():
    made = pools(1, "bf16", 2, 16, 1, 64, "token")
    before = made[0][0].clone()
    paged_move([describe(*made[0], "bf16")], torch.zeros(0, 4, dtype=torch.int32, device="cuda"),
               torch.zeros(0, 4, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(made[0][0], before)
