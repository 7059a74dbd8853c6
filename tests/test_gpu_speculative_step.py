"""Steps of a server that drafts: a model of two layers, its requests' trees and prompts verified at once.  What stands is
compared with the same model run token by token in 64 bits: keys and values of every kept token where the tables say,
its logits, and the tokens that come out."""
import numpy as np
import pytest
import torch

from paged_common import describe, half_step, lib, make_cache, native, paged_qkv, rope_words, sample, stream
from speculate_common import at, attend_tree, controls, paged_accept, paged_move, paged_tree, put, tree64

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, DIM, PAGE, VOCAB = 96, 4, 1, 64, 8, 200
ROWS, WIDTH, PAGES, CAPACITY, LAYERS, NODES, WORDS = 4, 14, 56, 90, 2, 8, 2


class Server:
    def __init__(self, kind):
        g = torch.Generator("cuda").manual_seed(5)
        random = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
        zeros = lambda *shape, fill=0: torch.full(shape, fill, dtype=torch.int32, device="cuda")  # noqa: E731
        self.kind = kind
        self.caches = [make_cache(kind, PAGES, PAGE, KV, DIM) for _ in range(LAYERS)]
        t = self.caches[0][0].dtype
        wide = (HEADS + 2 * KV) * DIM
        self.embed, self.head = random(VOCAB, HIDDEN), random(HIDDEN, VOCAB) * HIDDEN ** -0.5 * 3
        self.into = [random(HIDDEN, wide) * HIDDEN ** -0.5 for _ in range(LAYERS)]
        self.back = [random(HEADS * DIM, HIDDEN) * (HEADS * DIM) ** -0.5 for _ in range(LAYERS)]
        self.gains = [(random(2, DIM) * 0.1).to(t) for _ in range(LAYERS)]
        self.words, self.cos, self.sin = rope_words(WIDTH * PAGE, DIM // 2)
        self.rope = self.words.cuda()
        self.lengths, self.counts, self.tables = zeros(ROWS), zeros(ROWS), zeros(ROWS, WIDTH, fill=-1)
        self.free, self.free_count = torch.randperm(PAGES, generator=g, device="cuda").int(), zeros(1, fill=PAGES)
        self.s = dict(lengths=self.lengths, offsets=zeros(ROWS + 1), parents=zeros(CAPACITY), tokens=zeros(CAPACITY),
                      drawn=zeros(CAPACITY + 1), given=zeros(ROWS), tables=self.tables, free=self.free, free_count=self.free_count,
                      lengths_out=self.lengths, free_out=self.free_count, accepted=zeros(ROWS, NODES + 1),
                      accepted_counts=zeros(ROWS), last=zeros(ROWS), status=zeros(1), **{"from": zeros(ROWS, NODES), "to": zeros(ROWS, NODES)})
        self.slots, self.places, self.table_status = zeros(CAPACITY), zeros(CAPACITY), zeros(1)
        self.positions, self.ancestors = zeros(CAPACITY), zeros(CAPACITY, WORDS)
        self.qkv = [torch.zeros(CAPACITY, wide, device="cuda") for _ in range(LAYERS)]
        self.q = torch.zeros(CAPACITY, HEADS * DIM, dtype=t, device="cuda")
        self.out = torch.zeros(CAPACITY, HEADS * DIM, dtype=t, device="cuda")
        self.logits, self.controlled = (torch.zeros(CAPACITY, VOCAB, device="cuda") for _ in range(2))
        self.history, self.said = zeros(ROWS, 300), zeros(ROWS)
        self.frequency = torch.full((ROWS,), 0.7, device="cuda")
        self.uniform, self.cold = torch.zeros(CAPACITY, device="cuda"), torch.zeros(CAPACITY, device="cuda")
        self.work = torch.empty(lib().plamo_kernel_attention_paged_tree_workspace(ROWS, CAPACITY, HEADS, KV, DIM), dtype=torch.uint8,
                                device="cuda")

    def launch(self):
        s = self.s
        native.call(lib().plamo_kernel_paged_tables, at(self.lengths), at(self.counts), ROWS, at(self.tables), WIDTH, PAGE,
                    at(self.free), at(self.free_count), PAGES, at(self.lengths), at(self.free_count), at(s["offsets"]),
                    at(self.slots), at(self.places), CAPACITY, at(self.table_status), stream())
        paged_tree(self.lengths, s["offsets"], s["parents"], CAPACITY, WORDS, 0, self.positions, self.ancestors)
        x = self.embed[s["tokens"].long()]
        for layer, (keys, values) in enumerate(self.caches):
            cache, gains = describe(keys, values, self.kind), self.gains[layer]
            torch.matmul(x, self.into[layer], out=self.qkv[layer])
            paged_qkv(cache, self.kind, self.qkv[layer], HEADS, self.slots, self.q, self.positions, gains[0], gains[1], self.rope)
            attend_tree(cache, self.q, HEADS, self.tables, self.lengths, s["offsets"], self.out, positions=self.positions,
                        ancestors=self.ancestors, workspace=self.work)
            x = x + self.out.float() @ self.back[layer]
        torch.matmul(x, self.head, out=self.logits)
        controls(self.logits, VOCAB, self.controlled, dict(
            history=self.history, history_lengths=self.said, offsets=s["offsets"], tokens=s["tokens"], ancestors=self.ancestors,
            frequency=self.frequency), ROWS)
        token, _ = sample(self.controlled, VOCAB, self.uniform, temperature=self.cold, prob=False, workspace=self.sample_work)
        s["drawn"].copy_(token)
        paged_accept(s, PAGE, NODES, PAGES)
        paged_move([describe(k, v, self.kind) for k, v in self.caches], s["from"], s["to"])

    sample_work = None

    # ---- the model token by token, in 64 bits
    def model(self, tokens, positions):
        """Logits, and per layer the keys and values, of a sequence of tokens."""
        x = self.embed.double().cpu()[tokens]
        stored = []
        for layer in range(LAYERS):
            rows = (x @ self.into[layer].double().cpu()).view(len(tokens), HEADS + 2 * KV, DIM)
            g = 1 + torch.cat([self.gains[layer][0].double().cpu().expand(HEADS, DIM), self.gains[layer][1].double().cpu().expand(KV, DIM)])
            turn = rows[:, :HEADS + KV]
            turn = turn / torch.sqrt((turn ** 2).mean(-1, keepdim=True) + 1e-6) * g
            c, s = self.cos[positions][:, None], self.sin[positions][:, None]
            a, b = turn[..., :DIM // 2], turn[..., DIM // 2:]
            turn = torch.cat([a * c - b * s, b * c + a * s], -1)
            k, v = turn[:, HEADS:], rows[:, HEADS + KV:]
            stored.append((k, v))
            score = torch.einsum("ihd,jd->hij", turn[:, :HEADS], k[:, 0]) / DIM ** 0.5
            score = score.masked_fill(torch.ones(len(tokens), len(tokens)).triu(1).bool(), float("-inf"))
            out = torch.einsum("hij,jd->ihd", torch.softmax(score, -1), v[:, 0]).reshape(len(tokens), -1)
            x = x + out @ self.back[layer].double().cpu()
        return x @ self.head.double().cpu(), stored


def drafts(rng, root, guess):
    """A tree of up to NODES drafts behind a request's next token: the model's own guess now and then, other tokens else."""
    tokens, parents, tips = [root], [-1], [0]
    for _ in range(int(rng.integers(0, NODES + 1))):
        parent = int(rng.choice(tips[-3:]))
        tokens.append(guess(tokens, parents, parent) if rng.random() < 0.6 else int(rng.integers(0, VOCAB)))
        parents.append(parent)
        tips.append(len(tokens) - 1)
    return tokens, parents


def run_steps(kind, captured):
    server, rng = Server(kind), np.random.default_rng(8)
    s = server.s
    sizes = lib().plamo_kernel_sample_workspace(CAPACITY, VOCAB)
    server.sample_work = torch.zeros(max(16, sizes), dtype=torch.uint8, device="cuda")
    texts = [rng.integers(0, VOCAB, n).tolist() for n in (30, 1, 12, 19)]  # what stands in the cache, or is to
    pending = [list(t) for t in texts]   # prompts, whole, come first
    standing = [[] for _ in range(ROWS)]
    said = [[] for _ in range(ROWS)]
    graph = None
    kept_drafts = 0
    for step in range(9):
        batch = []
        for r in range(ROWS):
            if step == 3 and r == 1:
                batch.append(([], [], 0, 0))   # rests for a step
            elif step == 5 and r == 2:
                batch.append(([], [], 0, -1))  # ends
                standing[r], said[r] = [], []
            elif not standing[r]:
                batch.append((pending[r], list(range(-1, len(pending[r]) - 1)), len(pending[r]), len(pending[r])))
            else:
                def guess(tokens, parents, parent, r=r):
                    line, at_node = [], parent
                    while at_node >= 0:
                        line.append(tokens[at_node])
                        at_node = parents[at_node]
                    text = standing[r] + line[::-1]
                    x = server.model(text, torch.arange(len(text)))[0][-1].numpy()
                    return int(np.argmax(x - 0.7 * np.bincount(said[r] + line, minlength=VOCAB)))
                tokens, parents = drafts(rng, pending[r][0], guess)
                batch.append((tokens, parents, 1, len(tokens)))
        flat = lambda i: sum((b[i] for b in batch), [])  # noqa: E731
        pad = [0] * (CAPACITY - len(flat(0)))
        for name, value in (("tokens", flat(0) + pad), ("parents", flat(1) + pad), ("given", [b[2] for b in batch])):
            s[name].copy_(torch.tensor(value, dtype=torch.int32))
        server.counts.copy_(torch.tensor([b[3] for b in batch], dtype=torch.int32))
        history = torch.zeros(ROWS, 300, dtype=torch.int32)
        for r, line in enumerate(said):
            history[r, :len(line)] = torch.tensor(line, dtype=torch.int32)
        server.history.copy_(history)
        server.said.copy_(torch.tensor([len(line) for line in said], dtype=torch.int32))
        if captured and step == 1:
            torch.cuda.synchronize()
            keep = {k: v.clone() for k, v in vars(server).items() if isinstance(v, torch.Tensor)}
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                server.launch()
            for k, v in keep.items():  # (a capture runs nothing)
                assert torch.equal(getattr(server, k), v) or not v.is_floating_point()
        graph.replay() if graph is not None else server.launch()
        torch.cuda.synchronize()
        assert server.table_status.item() == 0 and s["status"].item() == 0
        # ---- what came out, against the model
        offsets, accepted, number = s["offsets"].tolist(), s["accepted"].tolist(), s["accepted_counts"].tolist()
        lengths = [len(standing[r]) + max(0, b[3]) for r, b in enumerate(batch)]
        want_positions, want_bits = tree64(lengths, offsets, flat(1), CAPACITY, WORDS)
        assert np.array_equal(server.positions.cpu().numpy(), want_positions)
        assert np.array_equal(server.ancestors.cpu().numpy(), want_bits)
        for r, (tokens, parents, given, count) in enumerate(batch):
            if count <= 0:
                assert number[r] == 0 and (count == 0 or server.lengths[r].item() == 0)
                continue
            new = accepted[r][:number[r]]
            drafted, bonus = new[:-1], new[-1]
            kept_drafts += len(drafted)
            text = standing[r] + tokens[:given] + drafted
            assert server.lengths[r].item() == len(text) and s["last"][r].item() < offsets[r + 1]
            logits, stored = server.model(text, torch.arange(len(text)))
            # keys and values of the whole text, where the table says; rounding to the type, and what the layer before
            # carries on of it: a few dozen half steps of values of size 1 to 4
            half = half_step(kind)
            for layer, (keys, values) in enumerate(server.caches):
                where = torch.tensor([server.tables[r, j // PAGE].item() * PAGE + j % PAGE for j in range(len(text))]).cuda()
                for c, w in ((keys, stored[layer][0]), (values, stored[layer][1])):
                    got = c.reshape(-1, KV, DIM)[where].double().cpu()
                    assert (got - w).abs().max() <= half * (4 if layer == 0 else 64) + 1e-3, (step, r, layer)
            # each token that came out is the likeliest, or as likely as logits that are that far off can tell
            for i, token in enumerate(new):
                x = logits[len(text) - len(new) + i].numpy()
                line = said[r] + tokens[:given] + drafted[:i]
                x = x - 0.7 * np.bincount(line, minlength=VOCAB)
                assert x[token] >= x.max() - half * 256 - 1e-3, (step, r, i)
            standing[r], pending[r] = text, [bonus]
            said[r] = said[r] + tokens[:given] + drafted
        held = sum(-(-n // PAGE) for n in server.lengths.tolist())
        assert server.free_count.item() == PAGES - held
        live = [p for r in range(ROWS) for p in server.tables[r, :-(-server.lengths[r].item() // PAGE)].tolist()]
        assert sorted(live + server.free[:server.free_count.item()].tolist()) == list(range(PAGES))
    assert kept_drafts > 10  # the drafts were no idle ones


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_steps(kind):
    run_steps(kind, False)


def test_steps_on_one_graph():
    run_steps("bf16", True)
