"""Steps of a server with a model of two layers, prompts among them: the second layer's keys and values are of the
first layer's outputs, so every new token needs its attention, not a request's last one alone.  Attention takes a row a
new token: its request's table, and its position and the keys before it as the length.  Each layer is compared with
64 bits on the rows that it was given."""
import math

import numpy as np
import pytest
import torch

from paged_common import attend, describe, half_step, lib, make_cache, native, paged_qkv, qkv64, rope_words, stream

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, DIM, PAGE = 192, 6, 2, 64, 16
ROWS, WIDTH, PAGES, CAPACITY, LAYERS = 4, 12, 40, 130, 2


class Server:
    def __init__(self, kind):
        put = lambda *shape, fill=0: torch.full(shape, fill, dtype=torch.int32, device="cuda")  # noqa: E731
        g = torch.Generator("cuda").manual_seed(9)
        random = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
        self.kind = kind
        self.caches = [make_cache(kind, PAGES, PAGE, KV, DIM) for _ in range(LAYERS)]
        t = self.caches[0][0].dtype
        self.lengths, self.counts, self.tables = put(ROWS), put(ROWS), put(ROWS, WIDTH, fill=-1)
        self.free, self.free_count = torch.randperm(PAGES, generator=g, device="cuda").int(), put(1, fill=PAGES)
        self.offsets, self.slots, self.positions, self.status = put(ROWS + 1), put(CAPACITY), put(CAPACITY), put(1)
        self.x = torch.zeros(CAPACITY, HIDDEN, device="cuda")
        wide = (HEADS + 2 * KV) * DIM
        self.into = [random(HIDDEN, wide) * HIDDEN ** -0.5 for _ in range(LAYERS)]
        self.back = [random(HEADS * DIM, HIDDEN) * (HEADS * DIM) ** -0.5 for _ in range(LAYERS)]
        self.gains = [(random(2, DIM) * 0.1).to(t) for _ in range(LAYERS)]
        self.qkv = [torch.zeros(CAPACITY, wide, device="cuda") for _ in range(LAYERS)]
        # rows that no token writes stay NaN, and reach nothing
        self.q = torch.full((CAPACITY, HEADS * DIM), float("nan"), dtype=t, device="cuda")
        self.out = [torch.zeros(CAPACITY, HEADS * DIM, dtype=t, device="cuda") for _ in range(LAYERS)]
        self.words, self.cos, self.sin = rope_words(WIDTH * PAGE, DIM // 2)
        self.rope = self.words.cuda()
        self.places = torch.arange(CAPACITY, dtype=torch.int32, device="cuda")
        self.work = torch.empty(lib().plamo_kernel_attention_paged_workspace(CAPACITY, HEADS, KV, DIM), dtype=torch.uint8,
                                device="cuda")
        self.history = [[[] for _ in range(ROWS)] for _ in range(LAYERS)]

    def launch(self):
        at = lambda t: t.data_ptr()  # noqa: E731
        native.call(lib().plamo_kernel_paged_tables, at(self.lengths), at(self.counts), ROWS, at(self.tables), WIDTH, PAGE,
                    at(self.free), at(self.free_count), PAGES, at(self.lengths), at(self.free_count), at(self.offsets),
                    at(self.slots), at(self.positions), CAPACITY, at(self.status), stream())
        request = torch.searchsorted(self.offsets[1:], self.places, right=True).clamp(max=ROWS - 1)
        tables, visible = self.tables[request], self.positions + 1
        x = self.x
        for layer, (keys, values) in enumerate(self.caches):
            cache = describe(keys, values, self.kind)
            torch.matmul(x, self.into[layer], out=self.qkv[layer])
            gains = self.gains[layer]
            paged_qkv(cache, self.kind, self.qkv[layer], HEADS, self.slots, self.q, self.positions, gains[0], gains[1], self.rope)
            attend(cache, self.q, HEADS, tables, visible, self.out[layer], workspace=self.work)
            x = x + self.out[layer].float() @ self.back[layer]

    def step(self, counts, rng, launch):
        total = sum(max(0, c) for c in counts)
        self.counts.copy_(torch.tensor(counts, dtype=torch.int32))
        self.x.copy_(torch.from_numpy(rng.standard_normal(self.x.shape)))
        launch()
        torch.cuda.synchronize()
        assert self.status.item() == 0
        held = [len(h) for h in self.history[0]]
        positions = torch.tensor([n for h, c in zip(held, counts) for n in range(h, h + max(0, c))])
        assert self.positions.tolist() == positions.tolist() + [-1] * (CAPACITY - total)
        half = half_step(self.kind)
        for layer in range(LAYERS):
            rows, _ = qkv64(self.qkv[layer][:total], HEADS, KV, DIM, positions, self.cos, self.sin, self.gains[layer])
            assert torch.all(self.out[layer][total:] == 0)
            at = 0
            for r, c in enumerate(counts):
                if c < 0:
                    self.history[layer][r] = []
                for _ in range(max(0, c)):
                    own = self.history[layer][r]
                    own.append(rows[at])
                    stored = torch.stack(own)
                    group = torch.arange(HEADS) // (HEADS // KV)
                    k, v = stored[:, HEADS:HEADS + KV][:, group], stored[:, HEADS + KV:][:, group]
                    score = torch.einsum("hd,jhd->hj", rows[at, :HEADS], k) / math.sqrt(DIM)
                    share = torch.softmax(score, -1)
                    want = torch.einsum("hj,jhd->hd", share, v)
                    # queries, keys and values are rounded when they are stored, each half a step off; two roundings
                    # in a score, which a weight and the sum of the weights feel
                    most = (torch.einsum("hd,jhd->hj", rows[at, :HEADS].abs(), k.abs()) / math.sqrt(DIM)).amax(-1, keepdim=True)
                    slack = torch.einsum("hj,jhd->hd", share, v.abs()) * (half * (1 + 2 * 2 * most) + 1e-3) + want.abs() * half
                    got = self.out[layer][at].double().cpu().view(HEADS, DIM)
                    assert torch.all((got - want).abs() <= slack), (layer, r, len(own))
                    at += 1


STEPS = [[40, 1, 0, 17], [1, 1, 33, 1], [3, 0, 1, 25], [1, -1, 1, 1], [1, 70, -1, 0], [-1, 1, 50, 1]]


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_prompts_through_two_layers(kind):
    server, rng = Server(kind), np.random.default_rng(6)
    for counts in STEPS:
        server.step(counts, rng, server.launch)


def test_on_one_graph():
    server, rng = Server("bf16"), np.random.default_rng(7)
    server.step(STEPS[0], rng, server.launch)
    graph = torch.cuda.CUDAGraph()
    server.counts.zero_()
    with torch.cuda.graph(graph):
        server.launch()
    for counts in STEPS[1:]:
        server.step(counts, rng, graph.replay)
