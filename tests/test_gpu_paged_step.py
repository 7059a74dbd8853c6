"""The paged operators together, as a server runs them: tables, the projection's rows into the pages,
attention, and a drawn token, step after step, with requests that begin, wait and end.  The dense side
keeps every request's own keys and values and attends in 64 bits."""
import math

import numpy as np
import pytest
import torch

from paged_common import (attend, describe, half_step, lib, make_cache, native, paged_qkv, qkv64, rope_words, sample, sample64,
                          stream)

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, PAGE, VOCAB = 16, 1, 128, 16, 3001
ROWS, WIDTH, PAGES, CAPACITY = 5, 20, 60, 200


class Server:
    def __init__(self, kind):
        put = lambda *shape, fill=0: torch.full(shape, fill, dtype=torch.int32, device="cuda")  # noqa: E731
        self.kind = kind
        self.keys, self.values = make_cache(kind, PAGES, PAGE, KV, DIM, "joined")
        t = self.keys.dtype
        self.cache = describe(self.keys, self.values, kind)
        self.lengths, self.counts, self.tables = put(ROWS), put(ROWS), put(ROWS, WIDTH, fill=-1)
        self.free, self.free_count = torch.randperm(PAGES, device="cuda").int(), put(1, fill=PAGES)
        self.offsets, self.slots, self.positions, self.status = put(ROWS + 1), put(CAPACITY), put(CAPACITY), put(1)
        self.qkv = torch.zeros(CAPACITY, (HEADS + 2 * KV) * DIM, device="cuda")
        self.q = torch.zeros(CAPACITY, HEADS * DIM, dtype=t, device="cuda")
        self.last = torch.zeros(ROWS, HEADS * DIM, dtype=t, device="cuda")
        self.out = torch.zeros(ROWS, HEADS * DIM, dtype=t, device="cuda")
        self.gains = (torch.randn(2, DIM, device="cuda") * 0.1).to(t)
        self.words, self.cos, self.sin = rope_words(WIDTH * PAGE, DIM // 2)
        self.rope = self.words.cuda()
        self.head = torch.randn(HEADS * DIM, VOCAB, device="cuda") * 0.3
        self.logits = torch.zeros(ROWS, VOCAB, device="cuda")
        self.u, self.p = torch.zeros(ROWS, device="cuda"), torch.full((ROWS,), 0.9, device="cuda")
        self.work = torch.empty(lib().plamo_kernel_attention_paged_workspace(ROWS, HEADS, KV, DIM), dtype=torch.uint8,
                                device="cuda")
        self.sample_work = torch.empty(max(16, lib().plamo_kernel_sample_workspace(ROWS, VOCAB)), dtype=torch.uint8,
                                       device="cuda")
        self.history = [[] for _ in range(ROWS)]

    def launch(self):
        at = lambda t: t.data_ptr()  # noqa: E731
        native.call(lib().plamo_kernel_paged_tables, at(self.lengths), at(self.counts), ROWS, at(self.tables), WIDTH, PAGE,
                    at(self.free), at(self.free_count), PAGES, at(self.lengths), at(self.free_count), at(self.offsets),
                    at(self.slots), at(self.positions), CAPACITY, at(self.status), stream())
        paged_qkv(self.cache, self.kind, self.qkv, HEADS, self.slots, self.q, self.positions, self.gains[0], self.gains[1],
                  self.rope)
        # each request's last row asks; one without new tokens repeats some row, which nobody looks at
        self.last.copy_(self.q[(self.offsets[1:].long() - 1).clamp(min=0)])
        attend(self.cache, self.last, HEADS, self.tables, self.lengths, self.out, workspace=self.work)
        self.logits.copy_(self.out.float() @ self.head)
        self.token, self.prob = sample(self.logits, VOCAB, self.u, top_p=self.p, workspace=self.sample_work)

    def step(self, counts, rng, launch):
        total = sum(max(0, c) for c in counts)
        self.counts.copy_(torch.tensor(counts, dtype=torch.int32))
        self.qkv.copy_(torch.from_numpy(rng.standard_normal(self.qkv.shape)))
        self.u.copy_(torch.from_numpy(rng.random(ROWS)))
        launch()
        torch.cuda.synchronize()
        assert self.status.item() == 0
        positions = [n for h, c in zip(self.history, counts) for n in range(len(h), len(h) + max(0, c))]
        assert self.positions.tolist() == positions + [-1] * (CAPACITY - total)
        rows, _ = qkv64(self.qkv[:total], HEADS, KV, DIM, torch.tensor(positions), self.cos, self.sin, self.gains)
        at, step = 0, half_step(self.kind)
        for r, c in enumerate(counts):
            if c < 0:
                self.history[r] = []
            self.history[r] += [rows[at + i] for i in range(max(0, c))]
            at += max(0, c)
            if c <= 0:
                continue
            stored = torch.stack(self.history[r])
            k, v = stored[:, HEADS], stored[:, HEADS + KV]
            share = torch.softmax(stored[-1, :HEADS] @ k.T / math.sqrt(DIM), -1)
            want = share @ v
            # queries, keys and values are rounded when they are stored, each half a step off
            score = (stored[-1, :HEADS].abs() @ k.abs().T / math.sqrt(DIM)).amax(-1, keepdim=True)
            slack = (share @ v.abs()) * (step * (1 + 2 * 2 * score) + 1e-3) + want.abs() * step
            assert torch.all((self.out[r].double().cpu().view(HEADS, DIM) - want).abs() <= slack)
            token, prob = sample64(self.logits[r].double().cpu().numpy(), float(self.u[r]), top_p=float(self.p[r]))
            assert int(self.token[r]) == token and abs(float(self.prob[r]) - prob) <= 1e-6
        assert self.lengths.tolist() == [len(h) for h in self.history]


STEPS = [[40, 1, 0, 17, 100], [1, 1, 33, 1, 1], [1, 1, 1, 1, 1], [-1, 1, 1, -1, 1], [64, 1, 1, 0, 1], [1, 1, 1, 20, -1],
         [1, 1, 1, 1, 3], [1, 1, 1, 1, 1]]


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_a_server_step_by_step(kind):
    server, rng = Server(kind), np.random.default_rng(3)
    for counts in STEPS:
        server.step(counts, rng, server.launch)


def test_a_server_on_one_graph():
    server, rng = Server("bf16"), np.random.default_rng(4)
    server.step([7, 0, 2, 1, 30], rng, server.launch)
    graph = torch.cuda.CUDAGraph()
    server.counts.zero_()
    with torch.cuda.graph(graph):
        server.launch()
    for counts in STEPS[1:]:
        server.step(counts, rng, graph.replay)
