"""A speculative step over a shared pool of KV pages, operator by operator, as measurable cases.

Drafted tokens are verified in one pass: every request brings a tree of them (or a chunk of its prompt).  Positions and
ancestors of the trees' nodes, attention of all of them over the request's pages, penalties, biases and grammar masks
on their logits, the path that the drawn tokens agree with (lengths cut, pages given back), and the kept tokens' keys
and values moved together in every layer.  Head layouts, layers, vocabulary and context lengths are the PLaMo-3 0.8B
model's (16 query heads on one KV head of 128, 16 layers, 107,520 tokens, a 2,048-key window), beside generic ones.
"""
import ctypes
import math
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
VOCAB = 107520
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a busy server's requests with a small tree each
        {"name": "tree_step", "op": "tree", "rows": 64, "nodes": 8, "chunk": 0, "words": 1, "window": 0, "pad": 0},
        # large trees beside chunks of new prompts, whose far ancestors a window leaves out
        {"name": "tree_mixed", "op": "tree", "rows": 200, "nodes": 60, "chunk": 500, "words": 16, "window": 256, "pad": 100},
        # one request early in a translation: the smallest verification that a token waits for
        {"name": "verify_one", "op": "attend", "rows": 1, "lo": 343, "hi": 343, "nodes": 8, "chain": False, "heads": 16,
         "kv": 1, "dim": 128, "type": "bf16", "page": 16, "window": 0},
        # a batch of the model's requests of all lengths, trees of up to 24 nodes
        {"name": "verify_batch", "op": "attend", "rows": 64, "lo": 33, "hi": 8192, "nodes": 24, "chain": False, "heads": 16,
         "kv": 1, "dim": 128, "type": "bf16", "page": 64, "window": 0},
        # grouped heads of 64 in FP16, a sliding window, pages of an odd number of tokens
        {"name": "verify_window", "op": "attend", "rows": 48, "lo": 1000, "hi": 9001, "nodes": 13, "chain": False,
         "heads": 32, "kv": 8, "dim": 64, "type": "fp16", "page": 48, "window": 2048},
        # chunks of two long prompts behind most of the context
        {"name": "chunk_long", "op": "attend", "rows": 2, "lo": 28000, "hi": 30720, "nodes": 999, "chain": True, "heads": 16,
         "kv": 1, "dim": 128, "type": "bf16", "page": 64, "window": 0},
        # one request's next token, a long history, all penalties
        {"name": "controls_one", "op": "controls", "rows": 1, "nodes": 0, "vocab": VOCAB, "type": "bf16", "out": "fp32",
         "history": 2000, "ngram": 3, "bias": 0, "masks": 0},
        # the nodes of a batch's trees: each with its path behind the history, grammars for half of them
        {"name": "controls_tree", "op": "controls", "rows": 32, "nodes": 8, "vocab": VOCAB, "type": "bf16", "out": "bf16",
         "history": 700, "ngram": 2, "bias": 40, "masks": 16},
        # small trees of a busy server
        {"name": "accept_step", "op": "accept", "rows": 64, "nodes": 8, "chunk": 0, "lo": 17, "hi": 4096, "page": 16},
        # many requests, trees beside chunks of prompts
        {"name": "accept_mixed", "op": "accept", "rows": 1000, "nodes": 32, "chunk": 500, "lo": 1, "hi": 30000, "page": 64},
        # what a verified step moves in the model's 16 layers
        {"name": "move_step", "op": "move", "layers": 16, "groups": 64, "group": 7, "kv": 1, "dim": 128, "type": "bf16",
         "page": 16},
        # requests of 20,000 tokens in all copied whole, for several continuations of them
        {"name": "move_copy", "op": "move", "layers": 16, "groups": 20000, "group": 1, "kv": 1, "dim": 128, "type": "bf16",
         "page": 64},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["tree", "attend", "attend", "attend", "controls", "controls", "accept", "move"])
    if op == "tree":
        words = _log(rng, 1, 16)
        most = 32 * words
        return {"op": op, "rows": _log(rng, 1, 1000 if words < 4 else 200), "nodes": _log(rng, 1, min(most, 100)),
                "chunk": rng.choice([0, _log(rng, 1, most)]), "words": words, "window": rng.choice([0, _log(rng, 1, 2 * most)]),
                "pad": rng.choice([0, rng.randint(1, 300)])}
    if op == "attend":
        kv, dim, chain = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256]), rng.random() < 0.4
        heads = kv * rng.choice([1, 2, 3, 4, 7, 8, 16])
        nodes = _log(rng, 1, 1000 if chain else 64)
        rows = _log(rng, 1, max(1, min(64, 8000 // nodes)))
        hi = _log(rng, 1, max(1, min(60000, 700_000_000 // (rows * heads * nodes) * 64 // dim, (1 << 21) * 128 // (rows * kv * dim))))
        return {"op": op, "rows": rows, "lo": _log(rng, 1, hi) - 1, "hi": hi, "nodes": nodes, "chain": chain, "heads": heads,
                "kv": kv, "dim": dim, "type": rng.choice(["bf16", "fp16"]), "page": rng.choice([8, 16, 24, 64, 100, 256]),
                "window": rng.choice([0, 0, _log(rng, 1, 4096)])}
    if op == "controls":
        nodes = rng.choice([0, 0, _log(rng, 1, 40)])
        kind = rng.choice(["bf16", "fp16", "fp32"])
        return {"op": op, "rows": _log(rng, 1, 64 // max(1, nodes // 8)), "nodes": nodes,
                "vocab": rng.choice([VOCAB, _log(rng, 1000, 110000)]), "type": kind, "out": rng.choice([kind, "fp32"]),
                "history": _log(rng, 1, 8000), "ngram": rng.choice([0, 2, 3, 5]), "bias": rng.choice([0, _log(rng, 1, 300)]),
                "masks": rng.choice([0, rng.randint(1, 9)])}
    if op == "accept":
        hi = _log(rng, 20, 30000)
        return {"op": op, "rows": _log(rng, 1, 1000), "nodes": _log(rng, 1, 64), "chunk": rng.choice([0, _log(rng, 2, 500)]),
                "lo": _log(rng, 1, hi), "hi": hi, "page": rng.choice([8, 16, 24, 64, 100])}
    kv, dim, group = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256]), rng.choice([1, 1, rng.randint(2, 40)])
    layers = rng.choice([1, 2, 16, 24])
    tokens = _log(rng, 1, 20000 * 16 * 128 // (layers * kv * dim))
    return {"op": op, "layers": layers, "groups": max(1, tokens // group), "group": group, "kv": kv, "dim": dim,
            "type": rng.choice(["bf16", "fp16"]), "page": rng.choice([1, 16, 24, 64])}


# ------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Cached tokens spread evenly over their logarithm."""
    at = np.linspace(math.log(case["lo"] + 1), math.log(case["hi"] + 1), case["rows"])
    return np.rint(np.exp(at)).astype(np.int64) - 1


def _counts(case):
    """New tokens of each request: trees of up to `nodes`, every eighth a chunk of its prompt, every eleventh none."""
    counts = np.rint(np.linspace(case["nodes"], max(1, case["nodes"] // 3), case["rows"])).astype(np.int64)
    counts[5::11] = 0
    if case.get("chunk"):
        counts[3::8] = case["chunk"]
    return counts


def _is_chunk(case):
    chunk = np.zeros(case["rows"], dtype=bool)
    if case.get("chunk"):
        chunk[3::8] = True
    return chunk


def _parents(rng, counts, chunk):
    """A parent among the six nodes before, its index in the request; chains for chunks."""
    offsets = np.concatenate([[0], np.cumsum(counts)])
    row = np.repeat(np.arange(len(counts)), counts)
    node = np.arange(offsets[-1]) - offsets[row]
    back = 1 + (rng.random(len(node)) ** 2 * 6).astype(np.int64)
    back[chunk[row]] = 1
    return offsets, row, node, np.where(node == 0, -1, np.maximum(0, node - back))


def _tables(rng, held, width, pages):
    """Tables of pages in random order, -1 behind, and the pages that are left."""
    order = rng.permutation(pages)
    tables = np.full((len(held), width), -1, dtype=np.int64)
    tables[np.arange(width)[None, :] < held[:, None]] = order[: int(held.sum())]
    return tables, order[int(held.sum()):]


def _ancestors(parent, row, offsets, words):
    """Bits of each node's ancestors and itself, and their number, on the host."""
    n = len(parent)
    bits, depth = np.zeros((n, words), dtype=np.uint32), np.zeros(n, dtype=np.int64)
    node = np.arange(n) - offsets[row]
    for i in range(n):
        if parent[i] >= 0:
            at = offsets[row[i]] + parent[i]
            bits[i], depth[i] = bits[at], depth[at] + 1
        bits[i, node[i] // 32] |= np.uint32(1 << (node[i] % 32))
    return bits.view(np.int32).astype(np.int64), depth


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed) * 7919 + 29)
    rng = np.random.default_rng([31, int(seed)])
    state = {"case": dict(case), "stream": torch.cuda.current_stream().cuda_stream}
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32).cuda()  # noqa: E731
    {"tree": _prepare_tree, "attend": _prepare_attend, "controls": _prepare_controls, "accept": _prepare_accept,
     "move": _prepare_move}[case["op"]](state, case, g, rng, put)
    return state


def _prepare_tree(state, case, g, rng, put):
    order = rng.permutation(case["rows"])
    counts, chunk = _counts(case)[order], _is_chunk(case)[order]
    offsets, _, _, parent = _parents(rng, counts, chunk)
    tokens = int(offsets[-1]) + case["pad"]
    full = np.zeros(tokens, dtype=np.int64)
    full[: offsets[-1]] = parent
    state.update(lengths=put(counts + rng.integers(0, 5000, case["rows"])), offsets=put(offsets), parents=put(full),
                 positions=put(np.zeros(tokens)), ancestors=put(np.zeros((tokens, case["words"]))))


def _prepare_attend(state, case, g, rng, put):
    kind, rows, dim, page, kv = TYPES[case["type"]], case["rows"], case["dim"], case["page"], case["kv"]
    before, counts = _lengths(case)[rng.permutation(rows)], _counts(case)
    lengths = before + counts
    held = -(-lengths // page)
    pages = int(held.sum()) + 2
    tables, _ = _tables(rng, held, max(1, int(held.max())), pages)
    offsets, row, _, parent = _parents(rng, counts, np.full(rows, case["chain"]))
    tokens = int(offsets[-1])
    words = -(-int(counts.max()) // 32)
    if not case["chain"]:
        bits, depth = _ancestors(parent, row, offsets, words)
        state.update(ancestors=put(bits), positions=put(before[row] + depth))
    cache = torch.randn(2, pages, page, kv, dim, generator=g, device="cuda", dtype=kind)
    state.update(keys=cache[0], values=cache[1], tables=put(tables), lengths=put(lengths), offsets=put(offsets),
                 most=int(counts.max()), words=words,
                 q=torch.randn(tokens, case["heads"] * dim, generator=g, device="cuda").to(kind),
                 out=torch.zeros(tokens, case["heads"] * dim, dtype=kind, device="cuda"),
                 lse=torch.zeros(tokens, case["heads"], device="cuda"))


def _prepare_controls(state, case, g, rng, put):
    sequences, vocab, kind = case["rows"], case["vocab"], TYPES[case["type"]]
    few = rng.integers(0, vocab, (sequences, 60))  # a text's own words come again
    said = lambda *shape: np.take_along_axis(few, rng.integers(0, 60, (sequences, *shape)), 1)  # noqa: E731
    lengths = rng.integers(case["history"] // 2, case["history"] + 1, sequences)
    state.update(history=put(said(case["history"])), history_lengths=put(lengths))
    rows = sequences
    if case["nodes"]:
        counts = _counts(case)
        offsets, row, node, parent = _parents(rng, counts, np.zeros(sequences, dtype=bool))
        words = -(-int(counts.max()) // 32)
        rows = int(offsets[-1])
        state.update(offsets=put(offsets), tokens=put(said(int(counts.max()))[row, node]), most=int(counts.max()),
                     ancestors=put(_ancestors(parent, row, offsets, words)[0]), words=words)
    uniform = lambda lo, hi: lo + (hi - lo) * torch.rand(sequences, generator=g, device="cuda")  # noqa: E731
    on = torch.arange(sequences, device="cuda") % 7 != 6  # every seventh request asks for no penalty
    state.update(logits=(torch.randn(rows, vocab, generator=g, device="cuda") * 2.2).to(kind),
                 repetition=torch.where(on, uniform(1.0, 1.4), 1.0), presence=torch.where(on, uniform(0.0, 0.8), 0.0),
                 frequency=torch.where(on, uniform(0.0, 0.3), 0.0),
                 ngram=put(np.where(np.arange(sequences) % 5 != 4, case["ngram"], 0)),
                 out=torch.zeros(rows, vocab, dtype=TYPES[case["out"]], device="cuda"))
    if case["bias"]:
        width = case["bias"]
        ids = (rng.integers(0, vocab, (sequences, 1)) + np.arange(width) * max(1, vocab // width)) % vocab
        ids[np.arange(width)[None, :] >= rng.integers(width // 2, width + 1, (sequences, 1))] = -1
        state.update(bias_ids=put(ids), bias=torch.randn(sequences, width, generator=g, device="cuda") * 3)
    if case["masks"]:
        words = -(-vocab // 32)
        masks = rng.integers(0, 1 << 32, (case["masks"], words), dtype=np.uint32)
        masks[::2] &= rng.integers(0, 1 << 32, masks[::2].shape, dtype=np.uint32) & rng.integers(0, 1 << 32, masks[::2].shape, dtype=np.uint32)
        state.update(masks=put(masks.view(np.int32)), mask_rows=put(np.where(rng.random(rows) < 0.5, rng.integers(0, case["masks"], rows), -1)))


def _prepare_accept(state, case, g, rng, put):
    rows, page, nodes = case["rows"], case["page"], case["nodes"]
    order = rng.permutation(rows)
    counts, chunk = _counts(case)[order], _is_chunk(case)[order]
    before = _lengths(case)[rng.permutation(rows)]
    held = -(-(before + counts) // page)
    pages = int((-(-before // page) + -(-counts // page)).sum()) + 9  # enough for any order of the requests
    tables, left = _tables(rng, held, int(held.max()) + 1, pages)
    offsets, row, node, parent = _parents(rng, counts, chunk)
    free = np.full(pages, -1, dtype=np.int64)
    free[: len(left)] = left
    tokens = rng.integers(0, VOCAB, len(node))
    # the model agrees with a draft in two cases of three
    drawn = rng.integers(0, VOCAB, len(node))
    agreed = np.flatnonzero((parent >= 0) & (rng.random(len(node)) < 2 / 3))
    drawn[offsets[row[agreed]] + parent[agreed]] = tokens[agreed]
    state.update(lengths=put(before + counts), offsets=put(offsets), parents=put(parent), tokens=put(tokens), drawn=put(drawn),
                 given=put(np.where(chunk, counts, 1)), tables=put(tables), free=put(free), free_count=put([len(left)]),
                 lengths_out=put(np.zeros(rows)), free_out=put([0]), accepted=put(np.zeros((rows, nodes + 1))),
                 accepted_counts=put(np.zeros(rows)), last=put(np.zeros(rows)), source=put(np.zeros((rows, nodes))),
                 target=put(np.zeros((rows, nodes))), status=put([0]), most=int(counts.max()))


def _prepare_move(state, case, g, rng, put):
    kind, page, groups, group = TYPES[case["type"]], case["page"], case["groups"], case["group"]
    pages = -(-(groups * (2 if group == 1 else group + 1)) // page) + 2
    if group == 1:  # from anywhere to slots that nothing is read from
        slots = rng.permutation(pages * page)[: 2 * groups].reshape(2, groups)
        source, target = slots[0][:, None], slots[1][:, None]
    else:  # the kept nodes of each request's `group + 1` to the places behind its first
        slots = rng.permutation(pages * page)[: groups * (group + 1)].reshape(groups, group + 1)
        kept = rng.random((groups, group)) < 0.5
        path = np.where(kept, np.arange(1, group + 1), 0)
        path = np.sort(np.where(path == 0, 1 << 20, path), 1)
        there = (path < 1 << 20) & (path != np.arange(1, group + 1))
        source = np.where(there, np.take_along_axis(slots, np.minimum(path, group), 1), -1)
        target = np.where(there, slots[:, 1:], -1)
    state.update(cache=torch.randn(case["layers"], 2, pages, page, case["kv"], case["dim"], generator=g, device="cuda",
                                   dtype=kind), source=put(source), target=put(target))


# ------------------------------------------------------------------------------ one pass
def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _spread(offsets, most):
    """Where request r's node i lies in the step, and whether it is there: [rows][most]."""
    first, count = offsets[:-1].long()[:, None], (offsets[1:] - offsets[:-1]).long()[:, None]
    node = torch.arange(most, device="cuda")[None, :]
    return torch.where(node < count, first + node, 0), node < count


def _reach(parents, there):
    """[rows][most][most]: whether node j is i or one of i's ancestors."""
    most = parents.shape[1]
    node = torch.arange(most, device="cuda")
    up = (there[..., None] & (parents[..., None] == node)).float()
    reach = up + torch.eye(most, device="cuda")
    for _ in range(max(1, most - 1).bit_length()):
        reach = (torch.matmul(reach, reach) > 0).float()
    return reach > 0


def _plain_tree(s):
    case, words = s["case"], s["case"]["words"]
    tokens, most = s["parents"].numel(), words * 32
    at, there = _spread(s["offsets"], most)
    reach = _reach(s["parents"].long()[at], there) & there[..., None]
    depth = reach.sum(-1) - 1
    if case["window"]:
        reach = reach & (depth[:, :, None] - depth[:, None, :] < case["window"])
    bits = (reach.long().view(*reach.shape[:2], words, 32) << torch.arange(32, device="cuda")).sum(-1)
    start = (s["lengths"] - (s["offsets"][1:] - s["offsets"][:-1])).long()[:, None]
    to = torch.where(there, at, tokens).reshape(-1)
    positions = torch.full((tokens + 1,), -1, device="cuda").index_put((to,), (start + depth).reshape(-1))
    ancestors = torch.zeros(tokens + 1, words, dtype=torch.int64, device="cuda").index_put((to,), bits.reshape(-1, words))
    s["positions"].copy_(positions[:tokens])
    s["ancestors"].copy_(torch.where(ancestors >= 1 << 31, ancestors - (1 << 32), ancestors)[:tokens])
    return {"positions": s["positions"], "ancestors": s["ancestors"]}


def _plain_attend(s):
    case = s["case"]
    rows, heads, kv, dim, page, most = case["rows"], case["heads"], case["kv"], case["dim"], case["page"], s["most"]
    group, width = heads // kv, s["tables"].shape[1]
    at, there = _spread(s["offsets"], most)
    start = (s["lengths"] - (s["offsets"][1:] - s["offsets"][:-1])).long()[:, None, None]
    key = torch.arange(width * page, device="cuda")[None, None, :]
    node = torch.arange(most, device="cuda")[None, :, None]
    new = key - start  # [rows][1][keys]: which new token a key is of
    if case["chain"]:
        position = start + node
        seen = key <= position
        if case["window"]:
            seen = seen & (key > position - case["window"])
    else:
        position = s["positions"].long()[at][..., None]
        words = s["ancestors"].long()[at]
        word = words.gather(2, (new.clamp(0, 32 * s["words"] - 1) // 32).expand(rows, most, -1))
        seen = (new >= 0) & (((word >> (new.clamp(min=0) % 32)) & 1) == 1)
        seen = seen | ((new < 0) & (key > position - case["window"] if case["window"] else new < 0))
    pages = s["tables"].long()[:, key[0, 0] // page]
    held = (key[0] < s["lengths"].long()[:, None]) & (pages >= 0)
    seen = seen & held[:, None] & there[..., None]
    pages = torch.where(held, pages, 0)
    k, v = (c[pages, key[0, 0] % page].float() for c in (s["keys"], s["values"]))  # [rows][keys][kv][dim]
    q = s["q"].float().view(-1, kv, group, dim)[at].permute(0, 2, 1, 3, 4).reshape(rows, kv, most * group, dim)
    score = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) / math.sqrt(dim)
    seen = seen[:, None, :, None, :].expand(rows, kv, most, group, -1).reshape(score.shape)
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(score - top)
    total = e.sum(-1, keepdim=True)
    v = torch.where(held[:, :, None, None], v, 0.0).permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(e, v) / torch.where(total == 0, 1.0, total)
    back = lambda x: x.view(rows, kv, most, group, -1).permute(0, 2, 1, 3, 4)[there]  # noqa: E731
    s["out"].copy_(back(out).reshape(-1, heads * dim))
    s["lse"].copy_(back(top + torch.log(total)).reshape(-1, heads))
    return {"out": s["out"], "lse": s["lse"]}


def _plain_controls(s):
    case, vocab = s["case"], s["case"]["vocab"]
    rows = s["logits"].shape[0]
    history, length = s["history"].long(), s["history_lengths"].long()
    sequence = torch.arange(rows, device="cuda")
    if case["nodes"]:
        sequence = torch.searchsorted(s["offsets"][1:].long(), sequence, right=True)
        # the path's tokens behind the history
        most = s["most"]
        node = torch.arange(most, device="cuda")
        on = ((s["ancestors"].long()[:, node // 32] >> (node % 32)) & 1) == 1
        path = s["tokens"].long()[(s["offsets"].long()[sequence][:, None] + node).clamp(max=rows - 1)]
        place = torch.where(on, length[sequence][:, None] + on.long().cumsum(1) - 1, history.shape[1] + most)
        history = torch.nn.functional.pad(history[sequence], (0, most + 1)).scatter(1, place, path)[:, :-1]
        length = length[sequence] + on.sum(1)
    where = torch.arange(history.shape[1], device="cuda")[None, :]
    counts = torch.zeros(rows, vocab + 1, device="cuda")
    counts.scatter_add_(1, torch.where(where < length[:, None], history, vocab), torch.ones_like(history, dtype=torch.float32))
    count = counts[:, :vocab]
    per = lambda name: s[name].float()[sequence][:, None]  # noqa: E731
    x = s["logits"].float()
    y = torch.where(x > 0, x / per("repetition"), x * per("repetition")) - per("presence") - per("frequency") * count
    x = torch.where(count > 0, y, x)
    if case["bias"]:
        ids = s["bias_ids"].long()[sequence]
        add = torch.zeros(rows, vocab + 1, device="cuda").scatter(1, torch.where(ids < 0, vocab, ids), s["bias"][sequence])
        x = x + add[:, :vocab]
    banned = torch.zeros(rows, vocab + 1, device="cuda")
    if case["ngram"] > 1:
        span = s["ngram"].long()[sequence][:, None] - 1
        step = torch.arange(case["ngram"] - 1, device="cuda")[None, None, :]
        last = (length[:, None] - span).clamp(min=0)
        tail = history.gather(1, (last + step[0]).clamp(max=history.shape[1] - 1))
        begin = where[:, :, None] + step
        window = history[:, begin.clamp(max=history.shape[1] - 1).view(-1)].view(rows, -1, step.shape[2])
        same = ((window == tail[:, None, :]) | (step >= span[..., None])).all(-1) & (span > 0) & (where + span < length[:, None])
        follow = history.gather(1, (where + span.clamp(min=0)).clamp(max=history.shape[1] - 1))
        banned.scatter_(1, torch.where(same, follow, vocab), 1.0)
    x = torch.where(banned[:, :vocab] > 0, -math.inf, x)
    if case["masks"]:
        token = torch.arange(vocab, device="cuda")
        allowed = ((s["masks"].long()[:, token // 32] >> (token % 32)) & 1) == 1
        own_mask = s["mask_rows"].long()
        x = torch.where((own_mask[:, None] < 0) | allowed[own_mask.clamp(min=0)], x, -math.inf)
    s["out"].copy_(x)
    return {"out": s["out"]}


def _accept_out(s):
    return {k: s[k] for k in ("lengths_out", "free", "free_out", "accepted", "accepted_counts", "last", "source", "target", "status")}


def _plain_accept(s):
    case, most, nodes, page = s["case"], s["most"], s["case"]["nodes"], s["case"]["page"]
    rows, pages, width = case["rows"], s["free"].numel(), s["tables"].shape[1]
    at, there = _spread(s["offsets"], most)
    node = torch.arange(most, device="cuda")[None, :]
    count = there.sum(1, keepdim=True)
    given = torch.minimum(s["given"].long()[:, None].clamp(min=1), count)
    parent, token, drawn = (torch.where(there, s[k].long()[at], -1) for k in ("parents", "tokens", "drawn"))
    up = drawn.gather(1, parent.clamp(min=0))
    agrees = there & (node >= given) & (parent >= given - 1) & (up >= 0) & (token == up)
    # the first of siblings that all agree
    first = torch.full((rows, most), most, device="cuda").scatter_reduce(
        1, parent.clamp(min=0), torch.where(agrees, node.expand(rows, most), most), "amin")
    fine = (agrees & (first.gather(1, parent.clamp(min=0)) == node)) | (there & (node < given))
    wrong = torch.matmul(_reach(parent, there).float(), (~fine).float()[..., None])[..., 0]
    kept = there & (fine & (wrong == 0) | (node < given))
    number = kept.sum(1, keepdim=True)
    path = torch.where(kept, node, most + node).sort(1).values  # kept nodes first
    final = path.gather(1, (number - 1).clamp(min=0))
    place = given + torch.arange(nodes, device="cuda")[None, :]
    more = place < number
    from_ = torch.nn.functional.pad(path, (0, nodes + 1)).gather(1, place.clamp(max=most + nodes))
    start = s["lengths"].long()[:, None] - count
    table = s["tables"].long()

    def slot(t):
        return table.gather(1, (t // page).clamp(0, width - 1)) * page + t % page
    moved = more & (from_ != place)
    s["source"].copy_(torch.where(moved, slot(start + from_), -1))
    s["target"].copy_(torch.where(moved, slot(start + place), -1))
    drafts = torch.where(more, token.gather(1, from_.clamp(max=most - 1)), -1)
    accepted = torch.nn.functional.pad(drafts, (0, 1), value=-1)
    some = count > 0
    end = (number - given).clamp(min=0)
    accepted = accepted.scatter(1, end, torch.where(some, drawn.gather(1, final.clamp(max=most - 1)), -1))
    s["accepted"].copy_(accepted)
    s["accepted_counts"].copy_(torch.where(some, end + 1, 0)[:, 0])
    s["last"].copy_(torch.where(some, s["offsets"][:-1].long()[:, None] + final, -1)[:, 0])
    length = start + number
    held, after = (s["lengths"].long()[:, None] + page - 1) // page, (length + page - 1) // page
    back = held - after
    column = torch.arange(width, device="cuda")[None, :]
    top = s["free_count"].long()
    to = torch.where((column >= after) & (column < held), top + back.cumsum(0) - back + column - after, pages)
    free = torch.cat([s["free"].long(), top * 0]).index_put((to.reshape(-1),), table.reshape(-1))
    s["free"].copy_(free[:pages])
    s["free_out"].copy_(top + back.sum())
    s["lengths_out"].copy_(length[:, 0])
    s["status"].zero_()
    return _accept_out(s)


def _plain_move(s):
    cache = s["cache"]
    flat = cache.view(cache.shape[0], 2, -1, *cache.shape[4:])
    source, target = s["source"].reshape(-1).long(), s["target"].reshape(-1).long()
    there = source >= 0
    source, target = source[there], target[there]
    flat[:, :, target] = flat[:, :, source]
    return {"cache": cache}


_plain = {"tree": _plain_tree, "attend": _plain_attend, "controls": _plain_controls, "accept": _plain_accept, "move": _plain_move}


# ------------------------------------------------------------------------------ the framework's calls
def _lib():
    if os.path.join(_ROOT, "plamo3-0.8b-runtime_amd") not in sys.path:
        sys.path.insert(0, os.path.join(_ROOT, "plamo3-0.8b-runtime_amd"))
    from plamo_hip import native
    return native


def _describe(native, keys, values, kind):
    return native.PagedCache(keys=keys.data_ptr(), values=values.data_ptr(), page_stride=keys.stride(0),
                             slot_stride=keys.stride(1), head_stride=keys.stride(2), pages=keys.shape[0],
                             page_size=keys.shape[1], kv_heads=keys.shape[2], head_dim=keys.shape[3], type=native.TYPES[kind])


def _handle(s):
    """What a program makes once and keeps: the library, the descriptions of its caches and controls, a workspace."""
    if "handle" in s:
        return s["handle"]
    native, case, what, work = _lib(), s["case"], None, None
    lib = native.load()
    at = lambda name: s[name].data_ptr() if name in s else 0  # noqa: E731
    if case["op"] == "attend":
        what = _describe(native, s["keys"], s["values"], case["type"])
        size = lib.plamo_kernel_attention_paged_tree_workspace(case["rows"], s["q"].shape[0], case["heads"], case["kv"], case["dim"])
        work = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
    if case["op"] == "move":
        what = (native.PagedCache * case["layers"])(*(_describe(native, c[0], c[1], case["type"]) for c in s["cache"]))
    if case["op"] == "controls":
        what = native.LogitControls(
            history=at("history"), history_lengths=at("history_lengths"), history_stride=s["history"].stride(0),
            sequences=case["rows"], history_width=s["history"].shape[1], offsets=at("offsets"), tokens=at("tokens"),
            ancestors=at("ancestors"), words=s.get("words", 0), repetition=at("repetition"), presence=at("presence"),
            frequency=at("frequency"), ngram=at("ngram"), bias_ids=at("bias_ids"), bias=at("bias"), bias_width=case["bias"],
            masks=at("masks"), mask_rows=at("mask_rows"), mask_stride=s["masks"].stride(0) if "masks" in s else 0,
            mask_count=case["masks"])
    s["handle"] = native, lib, what, work
    return s["handle"]


def _own_tree(s):
    native, lib, _, _ = _handle(s)
    native.call(lib.plamo_kernel_paged_tree, s["lengths"].data_ptr(), s["offsets"].data_ptr(), s["case"]["rows"],
                s["parents"].data_ptr(), s["parents"].numel(), s["case"]["window"], s["positions"].data_ptr(),
                s["ancestors"].data_ptr(), s["case"]["words"], s["stream"])
    return {"positions": s["positions"], "ancestors": s["ancestors"]}


def _own_attend(s):
    native, lib, cache, work = _handle(s)
    case, tree = s["case"], not s["case"]["chain"]
    native.call(lib.plamo_kernel_attention_paged_tree, cache, s["q"].data_ptr(), s["q"].stride(0), case["heads"],
                s["tables"].data_ptr(), s["tables"].shape[1], s["lengths"].data_ptr(), s["offsets"].data_ptr(), case["rows"],
                s["q"].shape[0], s["positions"].data_ptr() if tree else 0, s["ancestors"].data_ptr() if tree else 0,
                s["words"] if tree else 0, 1 / math.sqrt(case["dim"]), case["window"], s["out"].data_ptr(), s["out"].stride(0),
                s["lse"].data_ptr(), work.data_ptr(), work.numel(), s["stream"])
    return {"out": s["out"], "lse": s["lse"]}


def _own_controls(s):
    native, lib, controls, _ = _handle(s)
    case, logits = s["case"], s["logits"]
    native.call(lib.plamo_kernel_logit_controls, ctypes.byref(controls), logits.data_ptr(), native.TYPES[case["type"]],
                logits.stride(0), case["vocab"], logits.shape[0], s["out"].data_ptr(), native.TYPES[case["out"]],
                s["out"].stride(0), s["stream"])
    return {"out": s["out"]}


def _own_accept(s):
    native, lib, _, _ = _handle(s)
    case = s["case"]
    at = lambda *names: [s[n].data_ptr() for n in names]  # noqa: E731
    native.call(lib.plamo_kernel_paged_accept, *at("lengths", "offsets"), case["rows"], *at("parents", "tokens", "drawn"),
                s["parents"].numel(), *at("given", "tables"), s["tables"].shape[1], case["page"], *at("free", "free_count"),
                s["free"].numel(), *at("lengths_out", "free_out", "accepted", "accepted_counts", "last"), case["nodes"],
                *at("source", "target", "status"), s["stream"])
    return _accept_out(s)


def _own_move(s):
    native, lib, caches, _ = _handle(s)
    case = s["case"]
    native.call(lib.plamo_kernel_paged_move, caches, case["layers"], s["source"].data_ptr(), s["target"].data_ptr(),
                case["groups"], case["group"], s["stream"])
    return {"cache": s["cache"]}


_own = {"tree": _own_tree, "attend": _own_attend, "controls": _own_controls, "accept": _own_accept, "move": _own_move}


# ------------------------------------------------------------------------------ work
def work(case):
    if case["op"] == "tree":
        total = int(_counts(case).sum())
        return {"bytes": 8 * case["rows"] + 4 * total + 4 * (total + case["pad"]) * (1 + case["words"]), "flops": total * case["words"]}
    if case["op"] == "attend":
        before, counts = _lengths(case), _counts(case)
        wide, window = case["heads"] * case["dim"], case["window"]
        keys = counts.astype(np.float64) * 0 + np.where(counts > 0, np.minimum(before, window + counts) if window else before, 0)
        # scores: the cached keys of every new token, and about half of the new ones
        scores = float((counts * (np.minimum(before, window) if window else before) + counts * (counts + 1) / 2).sum())
        return {"bytes": float((keys + counts).sum()) * case["kv"] * case["dim"] * 4 + int(counts.sum()) * (4 * wide + 4 * case["heads"]),
                "flops": 4 * scores * wide}
    if case["op"] == "controls":
        rows = int(_counts(case).sum()) if case["nodes"] else case["rows"]
        size = {"bf16": 2, "fp16": 2, "fp32": 4}
        masks = case["masks"] * case["vocab"] // 8
        return {"bytes": rows * case["vocab"] * (size[case["type"]] + size[case["out"]]) + masks + 3 * case["rows"] * case["history"] +
                8 * case["rows"] * case["bias"], "flops": 2 * rows * case["vocab"]}
    if case["op"] == "accept":
        total = int(_counts(case).sum())
        return {"bytes": 12 * total + case["rows"] * (24 + 4 * (case["nodes"] + 1) + 8 * case["nodes"]), "flops": 2 * total}
    # about half of a group's nodes are kept, and most of these move
    tokens = case["groups"] if case["group"] == 1 else case["groups"] * case["group"] * 0.45
    return {"bytes": int(tokens * 2 * case["kv"] * case["dim"] * 2 * case["layers"] * 2) + 8 * case["groups"] * case["group"], "flops": 0}


# ------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    if case["op"] == "attend":
        return _exact_attend(prepare(case, seed))
    return {"tree": _exact_tree, "controls": _exact_controls, "accept": _exact_accept, "move": _exact_move}[case["op"]](
        prepare(case, seed))


def _exact_tree(s):
    """Node by node, from the parents' bits as whole numbers."""
    words, window = s["case"]["words"], s["case"]["window"]
    parents, offsets, lengths = (s[k].cpu().tolist() for k in ("parents", "offsets", "lengths"))
    positions, rows = [-1] * len(parents), [[0] * words for _ in parents]
    for r, (first, end) in enumerate(zip(offsets, offsets[1:])):
        lines = []
        for i in range(end - first):
            line = (lines[parents[first + i]] if parents[first + i] >= 0 else []) + [i]
            lines.append(line)
            positions[first + i] = lengths[r] - (end - first) + len(line) - 1
            bits = sum(1 << j for j in (line[-window:] if window else line))
            rows[first + i] = [(bits >> (32 * w)) & 0xFFFFFFFF for w in range(words)]
    ancestors = np.array(rows, dtype=np.uint32).reshape(len(parents), words).view(np.int32)
    return {"positions": torch.tensor(positions, dtype=torch.int32), "ancestors": torch.from_numpy(ancestors.copy())}


def _exact_attend(s):
    """Request by request, in blocks of its new tokens, over its own keys alone."""
    case = s["case"]
    kv, dim, page, window = case["kv"], case["dim"], case["page"], case["window"]
    group = case["heads"] // kv
    offsets, out, lse = s["offsets"].cpu().tolist(), [], []
    for r, n in enumerate(s["lengths"].cpu().tolist()):
        first, end = offsets[r], offsets[r + 1]
        before = n - (end - first)
        at = torch.arange(n, device="cuda")
        pages = s["tables"][r].long()[at // page]
        k, v = (c[pages, at % page].double() for c in (s["keys"], s["values"]))
        for t in range(first, end, 128):
            some = torch.arange(t, min(end, t + 128), device="cuda")
            if case["chain"]:
                far = (before + some - first)[:, None] - at
                seen = (far >= 0) & (far < window if window else far >= 0)
            else:
                line = torch.stack([(s["ancestors"][some, j // 32] >> (j % 32)) & 1 for j in range(end - first)], 1) != 0
                near = at[:before] > s["positions"][some].long()[:, None] - window if window else torch.ones(
                    len(some), before, dtype=torch.bool, device="cuda")
                seen = torch.cat([near, line], 1)
            q = s["q"][some].double().view(len(some), kv, group, dim)
            heads, norms = [], []
            for j in range(kv):
                score = (q[:, j].reshape(-1, dim) @ k[:, j].T * dim ** -0.5).view(len(some), group, n)
                score = torch.where(seen[:, None], score, -math.inf)
                norm = torch.logsumexp(score, -1)
                share = torch.where(seen[:, None], torch.exp(score - norm[..., None]), 0.0)
                heads.append((share.view(-1, n) @ v[:, j]).view(len(some), group, dim))
                norms.append(norm)
            out.append(torch.stack(heads, 1).reshape(len(some), -1))
            lse.append(torch.stack(norms, 1).reshape(len(some), -1))
    return {"out": torch.cat(out), "lse": torch.cat(lse)}


def _exact_controls(s):
    """Row by row on the host."""
    case, vocab = s["case"], s["case"]["vocab"]
    host = lambda name: s[name].cpu().numpy() if name in s else None  # noqa: E731
    history, lengths, ngram, offsets, tokens, bits = (host(n) for n in (
        "history", "history_lengths", "ngram", "offsets", "tokens", "ancestors"))
    ids, bias, masks, mask_rows = (host(n) for n in ("bias_ids", "bias", "masks", "mask_rows"))
    rep, pres, freq = (host(n).astype(np.float64) for n in ("repetition", "presence", "frequency"))
    logits, out = s["logits"].double().cpu().numpy(), np.empty(s["logits"].shape)
    for t, x in enumerate(logits):
        r, said = t, []
        if offsets is not None:
            r = int(np.searchsorted(offsets[1:], t, side="right"))
            said = [int(tokens[offsets[r] + j]) for j in range(offsets[r + 1] - offsets[r]) if bits[t, j // 32] >> (j % 32) & 1]
        said = history[r, : lengths[r]].tolist() + said
        x = x.copy()
        at, count = np.unique(np.array(said, dtype=np.int64), return_counts=True)
        x[at] = np.where(x[at] > 0, x[at] / rep[r], x[at] * rep[r]) - pres[r] - freq[r] * count
        if ids is not None:
            use = ids[r] >= 0
            x[ids[r][use]] += bias[r][use]
        span = int(ngram[r]) - 1
        if span > 0:
            tail = said[len(said) - span:]
            x[[said[i + span] for i in range(len(said) - span) if said[i:i + span] == tail]] = -np.inf
        if masks is not None and mask_rows[t] >= 0:
            open_ = np.unpackbits(masks[mask_rows[t]].view(np.uint8), bitorder="little")[:vocab].astype(bool)
            x[~open_] = -np.inf
        out[t] = x
    return {"out": torch.from_numpy(out)}


def _exact_accept(s):
    """One request after the other, on the host."""
    page, nodes, most = s["case"]["page"], s["case"]["nodes"], s["free"].numel()
    names = ("lengths", "offsets", "parents", "tokens", "drawn", "given", "tables", "free", "free_count")
    lengths, offsets, parents, tokens, drawn, given, tables, stack, top = (s[k].cpu().tolist() for k in names)
    stack, out = stack[: top[0]], {k: [] for k in ("lengths_out", "accepted", "accepted_counts", "last", "source", "target")}
    for r, (first, end) in enumerate(zip(offsets, offsets[1:])):
        n, length = end - first, lengths[r]
        fixed = min(max(1, given[r]), n)
        kept, new = list(range(fixed)), []
        while kept and drawn[first + kept[-1]] >= 0:
            fits = [i for i in range(kept[-1] + 1, n) if parents[first + i] == kept[-1] and tokens[first + i] == drawn[first + kept[-1]]]
            if not fits:
                break
            kept.append(fits[0])
        before = length - n
        slot = lambda t: tables[r][t // page] * page + t % page  # noqa: E731
        moves = [(slot(before + k), slot(before + j)) if k != j else (-1, -1) for j, k in enumerate(kept)][fixed:]
        moves += [(-1, -1)] * (nodes - len(moves))
        if kept:
            new = [tokens[first + k] for k in kept[fixed:]] + [drawn[first + kept[-1]]]
        after = before + len(kept)
        stack += tables[r][-(-after // page): -(-length // page)]
        for name, value in (("lengths_out", after), ("accepted", new + [-1] * (nodes + 1 - len(new))), ("accepted_counts", len(new)),
                            ("last", first + kept[-1] if kept else -1), ("source", [a for a, _ in moves]), ("target", [b for _, b in moves])):
            out[name].append(value)
    whole = lambda a: torch.tensor(a, dtype=torch.int32)  # noqa: E731
    free = s["free"].cpu().tolist()
    return {**{k: whole(v) for k, v in out.items()}, "free": whole(stack + free[len(stack):most]), "free_out": whole([len(stack)]),
            "status": whole([0])}


def _exact_move(s):
    """Move after move of each group, on whole rows of the pool."""
    cache = s["cache"].double()
    flat = cache.view(cache.shape[0], 2, -1, *cache.shape[4:])
    for step in range(s["source"].shape[1]):
        source, target = s["source"][:, step].long(), s["target"][:, step].long()
        there = torch.nonzero(target >= 0)[:, 0]
        flat[:, :, target[there]] = flat[:, :, source[there]].clone()
    return {"cache": cache}
