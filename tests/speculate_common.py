"""Plain implementations, in 64 bits or on whole numbers, of the operators of a speculative step, and calls of the
library's entry points on torch tensors."""
import ctypes
import math

import numpy as np
import torch

from paged_common import TYPES, lib, native, stream

at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731


def put(a, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a))).to(dtype).cuda()


# ------------------------------------------------------------------------------ trees
def random_parents(rng, count, reach=6):
    """A parent among the `reach` nodes before each, now and then none."""
    return [-1 if i == 0 or rng.random() < 0.05 else int(rng.integers(max(0, i - reach), i)) for i in range(count)]


def lines_of(parents):
    """Each node's path, itself last; parents that are no node before it are none."""
    lines = []
    for i, p in enumerate(parents):
        lines.append((lines[p] if 0 <= p < i else []) + [i])
    return lines


def tree64(lengths, offsets, parents, tokens, words, window=0):
    """positions [tokens], ancestors [tokens][words] as int32."""
    positions, bits = np.full(tokens, -1, np.int64), np.zeros((tokens, words), np.uint32)
    for r, (first, end) in enumerate(zip(offsets, offsets[1:])):
        n = end - first
        if n > 32 * words or lengths[r] < n:
            continue
        for i, line in enumerate(lines_of(parents[first:end])):
            positions[first + i] = lengths[r] - n + len(line) - 1
            for j in line[-window:] if window else line:
                bits[first + i, j // 32] |= np.uint32(1 << (j % 32))
    return positions.astype(np.int32), bits.view(np.int32)


def paged_tree(lengths, offsets, parents, tokens, words, window=0, positions=None, ancestors=None):
    if positions is None:
        positions = torch.full((tokens,), -77, dtype=torch.int32, device="cuda")
        ancestors = torch.full((tokens, words), -77, dtype=torch.int32, device="cuda")
    native.call(lib().plamo_kernel_paged_tree, at(lengths), at(offsets), offsets.numel() - 1, at(parents), tokens, window,
                at(positions), at(ancestors), words, stream())
    return positions, ancestors


# ------------------------------------------------------------------------------ attention
def attend_tree(cache, q, heads, tables, lengths, offsets, out, lse=None, positions=None, ancestors=None, scale=None, window=0,
                workspace=None, tokens=None):
    rows, tokens = tables.shape[0], q.shape[0] if tokens is None else tokens
    size = lib().plamo_kernel_attention_paged_tree_workspace(rows, tokens, heads, cache.kv_heads, cache.head_dim)
    if workspace is None:
        # of arbitrary contents: the call reads nothing that it has not written
        workspace = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
    native.call(lib().plamo_kernel_attention_paged_tree, cache, at(q), q.stride(0), heads, at(tables), tables.shape[1],
                at(lengths), at(offsets), rows, tokens, at(positions), at(ancestors),
                0 if ancestors is None else ancestors.shape[1], 1 / math.sqrt(cache.head_dim) if scale is None else scale,
                window, at(out), out.stride(0), at(lse), at(workspace), workspace.numel(), stream())
    return workspace


def attend_tree64(keys, values, q, tables, lengths, offsets, scale, positions=None, ancestors=None, window=0):
    """-> out [tokens][heads * dim], lse [tokens][heads] of the requests' tokens, and how far a kernel with FP32 sums
    may be off them before its last rounding (for both)."""
    weights = torch.finfo(keys.dtype).eps / 2  # of the weights' rounding to the type
    pages, page, kv, dim = keys.shape
    heads = q.shape[1] // dim
    total = int(offsets[-1])
    out, lse = torch.zeros(total, heads, dim, dtype=torch.float64), torch.full((total, heads), -math.inf, dtype=torch.float64)
    s_out, s_lse = torch.zeros_like(out), torch.zeros_like(lse)
    x = q[:total].double().cpu().view(total, heads, dim)
    for r in range(len(tables)):
        first, end = int(offsets[r]), int(offsets[r + 1])
        n, count = int(lengths[r]), end - first
        if count == 0 or n < count:
            continue
        start, n = n - count, min(n, tables.shape[1] * page)
        slots = [(int(tables[r][j // page]), j % page) if 0 <= tables[r][j // page] < pages else (-1, 0) for j in range(n)]
        there = torch.tensor([p >= 0 for p, _ in slots], dtype=torch.bool)
        where = torch.tensor([max(p, 0) for p, _ in slots], dtype=torch.long), torch.tensor([s for _, s in slots], dtype=torch.long)
        k, v = (c[where[0].to(c.device), where[1].to(c.device)].double().cpu() for c in (keys, values))
        key = torch.arange(n)
        for i in range(count):
            if ancestors is None:
                pos = start + i
                seen = key <= pos
                if window:
                    seen &= key > pos - window
            else:
                pos = int(positions[first + i])
                seen = key < start
                if window:
                    seen &= key > max(pos, start) - window
                for j in range(min(count, 32 * ancestors.shape[1])):
                    if start + j < n:
                        seen[start + j] = bool(int(ancestors[first + i][j // 32]) >> (j % 32) & 1)
                if pos < 0:
                    seen[:] = False
            seen &= there
            if not seen.any():
                continue
            for h in range(heads):
                g = h // (heads // kv)
                ks, vs = k[seen][:, g], v[seen][:, g]
                t = first + i
                score = (ks @ x[t, h]) * scale
                lse[t, h] = torch.logsumexp(score, 0)
                share = torch.exp(score - lse[t, h])
                out[t, h] = share @ vs
                # a score is a sum of `dim` products in FP32, scaled (2^-23 each: the sum may be truncated); the
                # exponential and its argument add 2^-21 of the largest score and of 1
                most = (ks.abs() @ x[t, h].abs()).max() * abs(scale)
                one = float(most) * (dim + 4) * 2.0 ** -23 + 2.0 ** -21 * (1 + float(score.abs().max()))
                # the sum of the weights is a chain of half the keys in each of two lanes (2^-24 each)
                sums = len(score) * 2.0 ** -25 + 2.0 ** -20
                # weights are off by twice a score's error (numerator and sum) and by half a step of the type where they are
                # rounded once: sum_j (p_j (1 + e_j) - p_j) v_j is at most max |e_j| sum_j p_j |v_j|; the products' sums are
                # chains of two steps for sixteen keys (2^-23 each: they may be truncated), and of the joins
                s_out[t, h] = (share @ vs.abs()) * (2 * one + sums + weights + (len(score) / 8 + 64) * 2.0 ** -23)
                s_lse[t, h] = one + sums + 2.0 ** -22 * abs(float(lse[t, h]))
    return out.view(total, -1), lse, s_out.view(total, -1), s_lse


# ------------------------------------------------------------------------------ controls
def controls(logits, n, out, spec, sequences):
    """`spec`: tensors by the fields' names."""
    c = native.LogitControls(sequences=sequences)
    for name, value in spec.items():
        setattr(c, name, at(value))
    if "history" in spec:
        c.history_stride, c.history_width = spec["history"].stride(0), spec["history"].shape[1]
    if "ancestors" in spec:
        c.words = spec["ancestors"].shape[1]
    if "bias_ids" in spec:
        c.bias_width = spec["bias_ids"].shape[1]
    if "masks" in spec:
        c.mask_stride, c.mask_count = spec["masks"].stride(0), spec["masks"].shape[0]
    names = {v: native.TYPES[k] for k, v in TYPES.items()}
    native.call(lib().plamo_kernel_logit_controls, ctypes.byref(c), at(logits), names[logits.dtype], logits.stride(0), n,
                logits.shape[0], at(out), names[out.dtype], out.stride(0), stream())


def controls64(x, said, repetition=1.0, presence=0.0, frequency=0.0, ngram=0, bias=(), mask=None):
    """One row (64-bit values) -> the row, and how far FP32 may be off it before its last rounding."""
    y, slack = np.array(x, np.float64), np.zeros(len(x))
    repetition = 1.0 if not repetition > 0 else repetition
    presence, frequency = (0.0 if math.isnan(v) else v for v in (presence, frequency))
    with np.errstate(all="ignore"):
        for token in set(said):
            if 0 <= token < len(y):
                count = said.count(token)
                z = y[token] / repetition if y[token] > 0 else y[token] * repetition
                y[token] = z - presence - frequency * count
                # a rounding of the product, of frequency's, and of the two differences
                slack[token] = 2.0 ** -24 * (3 * abs(z) + 2 * abs(presence) + 2 * abs(frequency) * count)
        for token, add in dict(bias).items():
            if 0 <= token < len(y):
                y[token] += add
                slack[token] += 2.0 ** -24 * abs(y[token]) + 2.0 ** -24 * slack[token]
    span = ngram - 1
    if span > 0 and len(said) >= ngram:
        tail = said[len(said) - span:]
        for i in range(len(said) - span):
            if said[i:i + span] == tail and 0 <= said[i + span] < len(y):
                y[said[i + span]] = -math.inf
    if mask is not None:
        y[~mask] = -math.inf
    return y, slack


# ------------------------------------------------------------------------------ accepted paths
ACCEPTED = ("lengths_out", "free_out", "accepted", "accepted_counts", "last", "from", "to", "status")


def accept_step(lengths, offsets, parents, tokens, drawn, given, tables, page, free, pages, nodes):
    """One request after the other, on lists; `free` (a stack) is changed in place.  Nothing changes with a status other
    than 0."""
    rows, width, capacity = len(lengths), len(tables[0]), len(parents)
    status, back, result = 0, [], {k: [] for k in ("lengths_out", "accepted", "accepted_counts", "last", "from", "to")}
    for r in range(rows):
        first, end = offsets[r], offsets[r + 1]
        n = end - first
        if not 0 <= first <= end <= capacity or lengths[r] < n:
            status |= 8
            continue
        fixed = min(max(1, given[r]), n)
        held = -(-lengths[r] // page)
        status |= (2 if held > width else 0) | (4 if n - fixed > nodes else 0)
        if status:
            continue
        kept = list(range(fixed))
        while kept and drawn[first + kept[-1]] >= 0:
            fits = [i for i in range(max(kept[-1] + 1, fixed), n)
                    if parents[first + i] == kept[-1] and tokens[first + i] == drawn[first + kept[-1]]]
            if not fits:
                break
            kept.append(fits[0])
        before = lengths[r] - n

        def slot(t):
            entry = tables[r][t // page]
            return entry * page + t % page if 0 <= entry < pages else -1
        moves = [(slot(before + k), slot(before + j)) if k != j else (-1, -1) for j, k in enumerate(kept)][fixed:]
        moves = [m if min(m) >= 0 else (-1, -1) for m in moves] + [(-1, -1)] * (nodes - len(moves))
        new = [tokens[first + k] for k in kept[fixed:]] + [drawn[first + kept[-1]]] if kept else []
        after = before + len(kept)
        back += [e for e in tables[r][-(-after // page):held] if 0 <= e < pages]
        for name, value in (("lengths_out", after), ("accepted", new + [-1] * (nodes + 1 - len(new))),
                            ("accepted_counts", len(new)), ("last", first + kept[-1] if kept else -1),
                            ("from", [a for a, _ in moves]), ("to", [b for _, b in moves])):
            result[name].append(value)
    if len(free) + len(back) > pages:
        status |= 8
    if status:
        none = {"lengths_out": list(lengths), "accepted": [[-1] * (nodes + 1)] * rows, "accepted_counts": [0] * rows,
                "last": [-1] * rows, "from": [[-1] * nodes] * rows, "to": [[-1] * nodes] * rows}
        return {**none, "free_out": len(free), "status": status}
    free += back
    return {**result, "free_out": len(free), "status": 0}


def paged_accept(s, page, nodes, pages):
    """`s`: tensors; outputs by ACCEPTED's names among them."""
    native.call(lib().plamo_kernel_paged_accept, at(s["lengths"]), at(s["offsets"]), s["lengths"].numel(), at(s["parents"]),
                at(s["tokens"]), at(s["drawn"]), s["parents"].numel(), at(s.get("given")), at(s["tables"]), s["tables"].shape[1],
                page, at(s["free"]), at(s["free_count"]), pages, at(s["lengths_out"]), at(s["free_out"]), at(s["accepted"]),
                at(s["accepted_counts"]), at(s["last"]), nodes, at(s["from"]), at(s["to"]), at(s["status"]), stream())


# ------------------------------------------------------------------------------ moves
def paged_move(caches, source, target):
    array = (native.PagedCache * len(caches))(*caches)
    groups, group = source.shape
    native.call(lib().plamo_kernel_paged_move, array, len(caches), at(source), at(target), groups, group, stream())
