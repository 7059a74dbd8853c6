"""A decode step over a shared pool of KV pages, operator by operator, as measurable cases.

Four operators in the order in which a serving loop runs them: block tables and slot maps from the
requests' lengths, the projection's rows normalised, rotated and written into the pages, attention of
one new token per request over its pages, and a token drawn from the logits, counted from the
likeliest on.  Head layouts, vocabulary and context lengths are the PLaMo-3 0.8B model's (16 query heads
on one KV head of 128, 107,520 tokens, a 2,048-key window), beside generic ones (grouped heads, a head
of 64 or 256, FP16, odd vocabularies).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
VOCAB = 107520
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # every request of a busy server decodes one token: a page is taken now and then
        {"name": "tables_step", "op": "tables", "rows": 64, "lo": 17, "hi": 4096, "page": 16, "new": 1, "chunk": 0,
         "capacity": 64},
        # a step that mixes decoding, chunks of new prompts and finished requests
        {"name": "tables_mixed", "op": "tables", "rows": 1000, "lo": 1, "hi": 30000, "page": 64, "new": 1, "chunk": 500,
         "capacity": 65536},
        # the model's projection rows of four decoding requests, as its GEMV leaves them (FP32)
        {"name": "qkv_step", "op": "qkv", "tokens": 4, "heads": 16, "kv": 1, "dim": 128, "type": "bf16", "source": "fp32",
         "page": 16, "norm": True},
        # a prefill chunk of several prompts, BF16 rows of the projection's GEMM
        {"name": "qkv_chunk", "op": "qkv", "tokens": 8192, "heads": 16, "kv": 1, "dim": 128, "type": "bf16",
         "source": "bf16", "page": 64, "norm": True},
        # one request early in a translation: the smallest call that a token waits for
        {"name": "attend_one", "op": "attend", "rows": 1, "lo": 343, "hi": 343, "heads": 16, "kv": 1, "dim": 128,
         "type": "bf16", "page": 16, "window": 0},
        # a full batch of the model's requests of all lengths
        {"name": "attend_ragged", "op": "attend", "rows": 128, "lo": 33, "hi": 16384, "heads": 16, "kv": 1, "dim": 128,
         "type": "bf16", "page": 64, "window": 0},
        # grouped heads of 64 in FP16, a sliding window, pages of an odd number of tokens
        {"name": "attend_window", "op": "attend", "rows": 48, "lo": 1000, "hi": 9001, "heads": 32, "kv": 8, "dim": 64,
         "type": "fp16", "page": 48, "window": 2048},
        # two very long documents
        {"name": "attend_long", "op": "attend", "rows": 2, "lo": 131072, "hi": 131072, "heads": 32, "kv": 4, "dim": 128,
         "type": "bf16", "page": 128, "window": 0},
        # one request's next token, all controls on
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": VOCAB, "type": "bf16", "mix": "all", "pad": 0},
        # a batch whose requests ask for different controls, some for none
        {"name": "sample_mixed", "op": "sample", "rows": 64, "vocab": VOCAB, "type": "bf16", "mix": "mixed", "pad": 0},
        # top-p alone on FP32 logits: no bound on how many tokens are kept
        {"name": "sample_top_p", "op": "sample", "rows": 128, "vocab": VOCAB, "type": "fp32", "mix": "top_p", "pad": 0},
        # an odd vocabulary in rows padded to another stride, min-p alone
        {"name": "sample_odd", "op": "sample", "rows": 7, "vocab": 50021, "type": "fp16", "mix": "min_p", "pad": 27},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["tables", "qkv", "attend", "attend", "sample", "sample"])
    if op == "tables":
        rows, chunk = _log(rng, 1, 1000), rng.choice([0, _log(rng, 2, 500)])
        hi = _log(rng, 20, 30000)
        case = {"op": op, "rows": rows, "lo": _log(rng, 1, hi), "hi": hi, "page": rng.choice([1, 8, 16, 24, 64, 100, 256]),
                "new": rng.randint(0, 2), "chunk": chunk, "capacity": 0}
        if case["page"] == 1:
            case["lo"], case["hi"] = min(case["lo"], 2000), min(hi, 2000)
        total = int(_counts(case).clip(0).sum())
        return dict(case, capacity=min(65536, total + rng.randint(0, 1 + total // 4) + 1))
    if op == "qkv":
        kv, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
        return {"op": op, "tokens": _log(rng, 1, 8192 // kv * 64 // dim), "heads": kv * rng.choice([1, 2, 4, 8, 16 // kv]),
                "kv": kv, "dim": dim, "type": rng.choice(["bf16", "fp16"]), "source": rng.choice(["fp32", "same"]),
                "page": rng.choice([1, 16, 24, 64]), "norm": rng.random() < 0.7}
    if op == "attend":
        kv, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
        rows = _log(rng, 1, 128)
        hi = _log(rng, 1, min(131072, (1 << 20) * 128 // (rows * kv * dim)))
        return {"op": op, "rows": rows, "lo": _log(rng, 1, hi), "hi": hi, "heads": kv * rng.choice([1, 2, 3, 4, 7, 8, 16]),
                "kv": kv, "dim": dim, "type": rng.choice(["bf16", "fp16"]), "page": rng.choice([8, 16, 24, 64, 128, 256]),
                "window": rng.choice([0, 0, _log(rng, 1, 4096)])}
    rows, kind = _log(rng, 1, 128), rng.choice(["bf16", "fp16", "fp32"])
    return {"op": op, "rows": rows, "vocab": rng.choice([VOCAB, _log(rng, 1000, 110000)]), "type": kind,
            "mix": rng.choice(["all", "mixed", "top_p", "top_k", "min_p", "plain"]), "pad": rng.choice([0, 0, 1, 8])}


# ------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Lengths spread evenly over their logarithm; which request has which goes by the seed."""
    at = np.linspace(math.log(case["lo"]), math.log(case["hi"]), case["rows"])
    return np.rint(np.exp(at)).astype(np.int64)


def _counts(case):
    """New tokens of each request: every eighth brings a chunk of its prompt, every eleventh has ended."""
    counts = np.full(case["rows"], case["new"], dtype=np.int64)
    if case["chunk"]:
        counts[::8] = case["chunk"]
        counts[5::11] = -1
    return counts


def _table_case(case):
    """lengths, counts, pages held and pages needed afterwards, table width, pages in all."""
    length, count, page = _lengths(case), _counts(case), case["page"]
    held = -(-length // page)
    after = np.where(count < 0, 0, -(-(length + count) // page))
    need = int(np.where(count < 0, 0, after - held).sum())
    width = int(max(held.max(), after.max())) + 1
    return length, count, held, after, width, int(held.sum()) + need + 3


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed) * 7919 + 17)
    rng = np.random.default_rng([23, int(seed)])
    state = {"case": dict(case), "stream": torch.cuda.current_stream().cuda_stream}
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32).cuda()  # noqa: E731
    if case["op"] == "tables":
        length, count, held, _, width, pages = _table_case(case)
        rows = case["rows"]
        order = rng.permutation(rows)
        length, count, held = length[order], count[order], held[order]
        shuffled = rng.permutation(pages)
        tables = np.full((rows, width), -1, dtype=np.int64)
        used = np.arange(width)[None, :] < held[:, None]
        tables[used] = shuffled[: int(held.sum())]
        free = np.full(pages, -1, dtype=np.int64)
        left = shuffled[int(held.sum()):]
        free[: len(left)] = left
        state.update(lengths=put(length), counts=put(count), tables=put(tables), free=put(free), free_count=put([len(left)]),
                     lengths_out=put(np.zeros(rows)), free_out=put([0]), offsets=put(np.zeros(rows + 1)),
                     slots=put(np.zeros(case["capacity"])), positions=put(np.zeros(case["capacity"])), status=put([0]))
        return state
    if case["op"] == "qkv":
        kind, tokens, dim, page = TYPES[case["type"]], case["tokens"], case["dim"], case["page"]
        source = kind if case["source"] == "same" else TYPES[case["source"]]
        heads = case["heads"] + 2 * case["kv"]
        pages = -(-tokens * 5 // 4 // page) + 1
        angle = torch.arange(4096, device="cuda", dtype=torch.float64)[:, None] * (
            10000.0 ** (-torch.arange(dim // 2, device="cuda", dtype=torch.float64) / (dim // 2)))
        bits = [f(angle).to(torch.bfloat16).view(torch.int16).to(torch.int32) & 0xFFFF for f in (torch.cos, torch.sin)]
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].to(torch.int32)
        positions = torch.randint(0, 4096, (tokens,), generator=g, device="cuda", dtype=torch.int32)
        cache = torch.randn(2, pages, page, case["kv"], dim, generator=g, device="cuda").to(kind)
        gains = (torch.randn(2, dim, generator=g, device="cuda") * 0.1).to(kind)
        state.update(qkv=torch.randn(tokens, heads * dim, generator=g, device="cuda").to(kind).to(source), keys=cache[0],
                     values=cache[1], slots=slots, positions=positions, rope=(bits[0] | (bits[1] << 16)).to(torch.int32),
                     gains=gains, q=torch.zeros(tokens, case["heads"] * dim, dtype=kind, device="cuda"))
        return state
    if case["op"] == "attend":
        kind, rows, dim, page, kv = TYPES[case["type"]], case["rows"], case["dim"], case["page"], case["kv"]
        length = _lengths(case)[rng.permutation(rows)]
        held = -(-length // page)
        width, pages = int(held.max()), int(held.sum()) + 2
        tables = np.full((rows, width), -1, dtype=np.int64)
        tables[np.arange(width)[None, :] < held[:, None]] = rng.permutation(pages)[: int(held.sum())]
        cache = torch.randn(2, pages, page, kv, dim, generator=g, device="cuda", dtype=kind)
        state.update(keys=cache[0], values=cache[1], tables=put(tables), lengths=put(length),
                     q=torch.randn(rows, case["heads"] * dim, generator=g, device="cuda").to(kind),
                     out=torch.zeros(rows, case["heads"] * dim, dtype=kind, device="cuda"),
                     lse=torch.zeros(rows, case["heads"], device="cuda"))
        return state
    rows, vocab, kind = case["rows"], case["vocab"], TYPES[case["type"]]
    # a bell of logits with some far above it, as a model's are
    logits = torch.randn(rows, vocab + case["pad"], generator=g, device="cuda") * 2.2
    likely = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")
    logits.scatter_add_(1, likely, torch.rand(rows, 24, generator=g, device="cuda") * 12)
    uniform = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, generator=g, device="cuda")  # noqa: E731
    row = torch.arange(rows, device="cuda")
    mix = case["mix"]
    on = lambda name, part: (row % 5 != part) if mix == "mixed" else (row >= 0) & (mix in ("all", name))  # noqa: E731
    temperature = torch.where((row % 9 == 8) & (mix == "mixed"), 0.0, uniform(0.6, 1.2))
    top_k = torch.where(on("top_k", 0), torch.randint(1, 200, (rows,), generator=g, device="cuda"), 0)
    top_p = torch.where(on("top_p", 1), uniform(0.6, 0.99), 1.0)
    min_p = torch.where(on("min_p", 2), uniform(0.005, 0.1), 0.0)
    state.update(logits=logits.to(kind)[:, :vocab], temperature=temperature, top_k=top_k.to(torch.int32), top_p=top_p,
                 min_p=min_p, uniform=torch.rand(rows, generator=g, device="cuda"),
                 token=torch.zeros(rows, dtype=torch.int32, device="cuda"), prob=torch.zeros(rows, device="cuda"))
    return state


# ------------------------------------------------------------------------------ one pass
def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _plain_tables(s):
    case = s["case"]
    page, capacity, pages = case["page"], case["capacity"], s["free"].numel()
    length, count, first = s["lengths"].long(), s["counts"].long(), s["free_count"].long()
    rows, width = s["tables"].shape
    ended = count < 0
    new = count.clamp(min=0)
    held = (length + page - 1) // page
    after = torch.where(ended, 0, (length + new + page - 1) // page)
    take = torch.where(ended, 0, after - held)
    back = torch.where(ended, held, 0)
    back_at, take_at = back.cumsum(0) - back, take.cumsum(0) - take
    full = first + back.sum()
    ends = new.cumsum(0)
    total = ends[-1:]
    status = ((take.sum() > full).long() + 2 * (after.amax() > width).long() + 4 * (total > capacity).long() +
              8 * (full > pages).long())
    fine = status == 0
    column = torch.arange(width, device="cuda")[None, :]
    old = s["tables"].long()
    # pages of the requests that ended, on top of the free ones (`pages`: a place for what is not written)
    at = torch.where(fine & ended[:, None] & (column < held[:, None]), first + back_at[:, None] + column, pages)
    free = torch.cat([s["free"].long(), first * 0]).index_put((at.reshape(-1),), old.reshape(-1))
    s["free"].copy_(free[:pages])
    fresh = fine & (column >= held[:, None]) & (column < after[:, None])
    from_ = (full - 1 - take_at[:, None] - (column - held[:, None])).clamp(0, pages - 1)
    s["tables"].copy_(torch.where(fresh, free[from_], old))
    s["lengths_out"].copy_(torch.where(fine, torch.where(ended, 0, length + new), length))
    s["free_out"].copy_(torch.where(fine, full - take.sum(), first))
    s["offsets"][1:].copy_(torch.where(fine, ends, 0))
    s["offsets"][:1].zero_()
    token = torch.arange(capacity, device="cuda")
    row = torch.searchsorted(ends, token, right=True).clamp(max=rows - 1)
    at = length[row] + token - (ends - new)[row]
    there = fine & (token < total)
    slot = s["tables"].long()[row, (at // page).clamp(0, width - 1)] * page + at % page
    s["slots"].copy_(torch.where(there, slot, -1))
    s["positions"].copy_(torch.where(there, at, -1))
    s["status"].copy_(status)
    return _tables_out(s)


def _tables_out(s):
    return {k: s[k] for k in ("tables", "free", "lengths_out", "free_out", "offsets", "slots", "positions", "status")}


def _plain_qkv(s):
    case = s["case"]
    tokens, heads, kv, dim, half = case["tokens"], case["heads"], case["kv"], case["dim"], case["dim"] // 2
    x = s["qkv"].float().view(tokens, heads + 2 * kv, dim)
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    if case["norm"]:
        gain = 1 + s["gains"].float()
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * gain[0]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * gain[1]
    pair = s["rope"][s["positions"].long()][:, None, :]
    cos, sin = (pair << 16).view(torch.float32), (pair & -65536).view(torch.float32)
    turn = lambda y: torch.cat([y[..., :half] * cos - y[..., half:] * sin, y[..., half:] * cos + y[..., :half] * sin], -1)  # noqa: E731
    s["q"].copy_(turn(q).reshape(tokens, -1))
    slot = s["slots"].long()
    pages, page = s["keys"].shape[:2]
    s["keys"].view(pages * page, kv, dim)[slot] = turn(k).to(s["keys"].dtype)
    s["values"].view(pages * page, kv, dim)[slot] = v.to(s["keys"].dtype)
    return {"q": s["q"], "keys": s["keys"], "values": s["values"]}


def _plain_attend(s):
    case = s["case"]
    rows, heads, kv, dim, page = case["rows"], case["heads"], case["kv"], case["dim"], case["page"]
    length, width = s["lengths"].long()[:, None], s["tables"].shape[1]
    at = torch.arange(width * page, device="cuda")
    first = (length - case["window"]).clamp(min=0) if case["window"] else length * 0
    pages = s["tables"].long()[:, at // page]
    seen = (at < length) & (at >= first) & (pages >= 0) & (pages < s["keys"].shape[0])
    pages = torch.where(seen, pages, 0)
    k, v = (c[pages, at % page].float() for c in (s["keys"], s["values"]))  # [rows][keys][kv][dim]
    q = s["q"].float().view(rows, kv, heads // kv, dim)
    score = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) / math.sqrt(dim)
    score = score.masked_fill(~seen[:, None, None, :], -math.inf)
    most = score.amax(-1, keepdim=True)
    most = torch.where(most == -math.inf, 0.0, most)
    e = torch.exp(score - most)
    total = e.sum(-1, keepdim=True)
    v = torch.where(seen[:, :, None, None], v, 0.0).permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(e, v) / torch.where(total == 0, 1.0, total)
    s["out"].copy_(out.reshape(rows, heads * dim))
    s["lse"].copy_((most + torch.log(total)).reshape(rows, heads))
    return {"out": s["out"], "lse": s["lse"]}


def _plain_sample(s):
    # in 64 bits: which token a number falls on is decided next to borders of long sums
    vocab = s["logits"].shape[1]
    x, token = torch.sort(torch.nan_to_num(s["logits"].double(), nan=-math.inf, posinf=math.inf, neginf=-math.inf), dim=1,
                          descending=True, stable=True)
    rank = torch.arange(vocab, device="cuda")[None, :]
    t = s["temperature"].double()[:, None]
    k = torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
    k = torch.where(t > 0, k, 1)
    top = x[:, :1]
    weight = torch.where(x == top, 1.0, torch.exp((x - top) / torch.where(t > 0, t, 1.0)))
    weight = torch.where((rank < k) & (x > -math.inf), weight, 0.0)
    sums = weight.cumsum(1)
    p = s["top_p"].double()[:, None]
    keep = (rank == 0) | (sums - weight < p * sums[:, -1:]) | (p >= 1)
    keep &= weight >= s["min_p"].double()[:, None].clamp(max=1)
    weight = torch.where(keep, weight, 0.0)
    sums = weight.cumsum(1)
    total = sums[:, -1:]
    last = torch.where(weight > 0, rank, 0).amax(1)
    at = torch.minimum((sums <= s["uniform"].double()[:, None].clamp(0, 1) * total).sum(1), last)[:, None]
    s["token"].copy_(token.gather(1, at)[:, 0])
    s["prob"].copy_((weight.gather(1, at) / total)[:, 0])
    return {"token": s["token"], "prob": s["prob"]}


_plain = {"tables": _plain_tables, "qkv": _plain_qkv, "attend": _plain_attend, "sample": _plain_sample}


# ------------------------------------------------------------------------------ the framework's calls
def _lib():
    if os.path.join(_ROOT, "plamo3-0.8b-runtime_amd") not in sys.path:
        sys.path.insert(0, os.path.join(_ROOT, "plamo3-0.8b-runtime_amd"))
    from plamo_hip import native
    return native


def _handle(s):
    """What a program makes once and keeps: the library, the description of its cache, a workspace."""
    if "handle" in s:
        return s["handle"]
    native, cache, work = _lib(), None, None
    case = s["case"]
    if "keys" in s:
        keys = s["keys"]
        cache = native.PagedCache(keys=keys.data_ptr(), values=s["values"].data_ptr(), page_stride=keys.stride(0),
                                  slot_stride=keys.stride(1), head_stride=keys.stride(2), pages=keys.shape[0],
                                  page_size=keys.shape[1], kv_heads=keys.shape[2], head_dim=keys.shape[3],
                                  type=native.TYPES[case["type"]])
    lib = native.load()
    size = 0
    if case["op"] == "attend":
        size = lib.plamo_kernel_attention_paged_workspace(case["rows"], case["heads"], case["kv"], case["dim"])
    if case["op"] == "sample":
        size = lib.plamo_kernel_sample_workspace(case["rows"], case["vocab"])
    work = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
    s["handle"] = native, lib, cache, work
    return s["handle"]


def _own_tables(s):
    native, lib, _, _ = _handle(s)
    rows, width = s["tables"].shape
    native.call(lib.plamo_kernel_paged_tables, s["lengths"].data_ptr(), s["counts"].data_ptr(), rows, s["tables"].data_ptr(),
                width, s["case"]["page"], s["free"].data_ptr(), s["free_count"].data_ptr(), s["free"].numel(),
                s["lengths_out"].data_ptr(), s["free_out"].data_ptr(), s["offsets"].data_ptr(), s["slots"].data_ptr(),
                s["positions"].data_ptr(), s["case"]["capacity"], s["status"].data_ptr(), s["stream"])
    return _tables_out(s)


def _own_qkv(s):
    native, lib, cache, _ = _handle(s)
    case = s["case"]
    source = case["type"] if case["source"] == "same" else case["source"]
    gains = (s["gains"][0].data_ptr(), s["gains"][1].data_ptr()) if case["norm"] else (0, 0)
    native.call(lib.plamo_kernel_paged_qkv, cache, s["qkv"].data_ptr(), native.TYPES[source], s["qkv"].stride(0),
                case["heads"], *gains, s["rope"].data_ptr(), s["rope"].shape[0], s["positions"].data_ptr(),
                s["slots"].data_ptr(), case["tokens"], s["q"].data_ptr(), s["q"].stride(0), s["stream"])
    return {"q": s["q"], "keys": s["keys"], "values": s["values"]}


def _own_attend(s):
    native, lib, cache, work = _handle(s)
    case = s["case"]
    native.call(lib.plamo_kernel_attention_paged, cache, s["q"].data_ptr(), s["q"].stride(0), case["heads"],
                s["tables"].data_ptr(), s["tables"].shape[1], s["lengths"].data_ptr(), case["rows"],
                1 / math.sqrt(case["dim"]), case["window"], s["out"].data_ptr(), s["out"].stride(0), s["lse"].data_ptr(),
                work.data_ptr(), work.numel(), s["stream"])
    return {"out": s["out"], "lse": s["lse"]}


def _own_sample(s):
    native, lib, _, work = _handle(s)
    case, logits = s["case"], s["logits"]
    native.call(lib.plamo_kernel_sample, logits.data_ptr(), native.TYPES[case["type"]], logits.stride(0), case["vocab"],
                case["rows"], s["temperature"].data_ptr(), s["top_k"].data_ptr(), s["top_p"].data_ptr(),
                s["min_p"].data_ptr(), s["uniform"].data_ptr(), s["token"].data_ptr(), s["prob"].data_ptr(),
                work.data_ptr(), work.numel(), s["stream"])
    return {"token": s["token"], "prob": s["prob"]}


_own = {"tables": _own_tables, "qkv": _own_qkv, "attend": _own_attend, "sample": _own_sample}


# ------------------------------------------------------------------------------ work
def work(case):
    if case["op"] == "tables":
        length, count, held, after, _, _ = _table_case(case)
        total = int(count.clip(0).sum())
        moved = int(np.where(count < 0, held, after - held).sum())  # a page id read and written for each
        # the entries that the new tokens lie in, lengths, counts, offsets, new lengths, both maps
        touched = int(np.where(count > 0, after - length // case["page"], 0).sum())
        return {"bytes": 16 * case["rows"] + 8 * moved + 4 * touched + 8 * case["capacity"] + 12, "flops": 4 * total}
    if case["op"] == "qkv":
        wide = case["heads"] + 2 * case["kv"]
        size = 4 if case["source"] == "fp32" else 2
        rope = 4 * min(case["tokens"], 4096) * case["dim"] // 2
        return {"bytes": case["tokens"] * (wide * case["dim"] * (size + 2) + 8) + rope,
                "flops": 7 * case["tokens"] * wide * case["dim"]}
    if case["op"] == "attend":
        length = _lengths(case)
        seen = int((np.minimum(length, case["window"]) if case["window"] else length).sum())
        row = case["rows"] * case["heads"] * (4 * case["dim"] + 4)
        return {"bytes": seen * case["kv"] * case["dim"] * 4 + row + 4 * (seen // case["page"] + 2 * case["rows"]),
                "flops": 4 * seen * case["heads"] * case["dim"]}
    size = 4 if case["type"] == "fp32" else 2
    return {"bytes": case["rows"] * (case["vocab"] * size + 28), "flops": 4 * case["rows"] * case["vocab"]}


# ------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    return {"tables": _exact_tables, "qkv": _exact_qkv, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](
        prepare(case, seed))


def _exact_tables(s):
    """One request after the other, on the host."""
    page, capacity = s["case"]["page"], s["case"]["capacity"]
    h = {k: s[k].cpu().tolist() for k in ("lengths", "counts", "tables", "free", "free_count")}
    stack, tables, lengths = h["free"], [list(r) for r in h["tables"]], list(h["lengths"])
    top, slots, positions, offsets = h["free_count"][0], [], [], [0]
    for r, count in enumerate(h["counts"]):
        if count < 0:
            for c in range(-(-lengths[r] // page)):
                stack[top] = tables[r][c]
                top += 1
            lengths[r] = 0
    for r, count in enumerate(h["counts"]):
        for _ in range(max(0, count)):
            n = lengths[r]
            if n % page == 0:
                top -= 1
                tables[r][n // page] = stack[top]
            slots.append(tables[r][n // page] * page + n % page)
            positions.append(n)
            lengths[r] = n + 1
        offsets.append(len(slots))
    pad = [-1] * (capacity - len(slots))
    whole = lambda a: torch.tensor(a, dtype=torch.int32)  # noqa: E731
    return {"tables": whole(tables), "free": whole(stack), "lengths_out": whole(lengths), "free_out": whole([top]),
            "offsets": whole(offsets), "slots": whole(slots + pad), "positions": whole(positions + pad), "status": whole([0])}


def _exact_qkv(s):
    case = s["case"]
    heads, kv, half = case["heads"], case["kv"], case["dim"] // 2
    rows = s["qkv"].double().reshape(case["tokens"], -1, case["dim"])
    table = s["rope"].cpu().numpy().view(np.uint32)[s["positions"].cpu().numpy()]
    unpack = lambda a: torch.from_numpy(a.view(np.float32).astype(np.float64)).cuda()[:, None]  # noqa: E731
    turn = torch.complex(unpack(np.left_shift(table, 16)), unpack(table & np.uint32(0xFFFF0000)))
    out = []
    for part, gain in ((rows[:, :heads], s["gains"][0]), (rows[:, heads:heads + kv], s["gains"][1])):
        if case["norm"]:
            part = part / torch.sqrt(torch.linalg.vector_norm(part, dim=-1, keepdim=True) ** 2 / case["dim"] + EPS)
            part = part + part * gain.double()
        z = torch.complex(part[..., :half].contiguous(), part[..., half:].contiguous()) * turn
        out.append(torch.cat([z.real, z.imag], -1))
    cache = {}
    slot = s["slots"].long()
    for name, new in (("keys", out[1]), ("values", rows[:, heads + kv:])):
        flat = s[name].double().reshape(-1, kv, case["dim"])
        flat[slot] = new
        cache[name] = flat.reshape(s[name].shape)
    return {"q": out[0].reshape(case["tokens"], -1), **cache}


def _exact_attend(s):
    """Request by request, over its own keys alone."""
    case = s["case"]
    kv, dim, page = case["kv"], case["dim"], case["page"]
    out, lse = [], []
    for r, n in enumerate(s["lengths"].cpu().tolist()):
        at = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device="cuda")
        pages = s["tables"][r].long()[at // page]
        k, v = s["keys"][pages, at % page].double(), s["values"][pages, at % page].double()
        q = s["q"][r].double().view(kv, -1, dim)
        score = torch.stack([q[j] @ k[:, j].T for j in range(kv)]) * dim ** -0.5
        norm = torch.logsumexp(score, -1)
        share = torch.exp(score - norm[..., None])
        out.append(torch.cat([(share[j] @ v[:, j]).reshape(-1) for j in range(kv)]))
        lse.append(norm.reshape(-1))
    return {"out": torch.stack(out), "lse": torch.stack(lse)}


def _exact_sample(s):
    """Row by row on the host, the kept tokens listed from the likeliest on."""
    logits = s["logits"].double().cpu().numpy()
    host = lambda name: s[name].double().cpu().numpy()  # noqa: E731
    temperature, top_k, top_p, min_p, uniform = (host(n) for n in ("temperature", "top_k", "top_p", "min_p", "uniform"))
    tokens, probs = [], []
    for r, x in enumerate(logits):
        if temperature[r] <= 0:
            tokens.append(int(np.argmax(x)))
            probs.append(1.0)
            continue
        order = np.argsort(-x, kind="stable")
        if top_k[r] > 0:
            order = order[: int(top_k[r])]
        w = np.exp((x[order] - x[order[0]]) / temperature[r])
        if top_p[r] < 1:
            before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            cut = np.flatnonzero(before >= top_p[r] * math.fsum(w))
            order = order[: max(1, int(cut[0]) if len(cut) else len(order))]
            w = w[: len(order)]
        order, w = order[w >= min_p[r]], w[w >= min_p[r]]
        sums = np.cumsum(w)
        at = min(int(np.searchsorted(sums, uniform[r] * sums[-1], side="right")), len(order) - 1)
        tokens.append(int(order[at]))
        probs.append(float(w[at] / sums[-1]))
    return {"token": torch.tensor(tokens, dtype=torch.int32), "prob": torch.tensor(probs, dtype=torch.float64)}
