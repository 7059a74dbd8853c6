"""Plain implementations, in 64 bits or on whole numbers, of the operators over paged caches and of the
sampler, and calls of the library's entry points on torch tensors."""
import math

import numpy as np
import torch

from plamo_hip import native

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def lib():
    return native.load()


def stream():
    return torch.cuda.current_stream().cuda_stream


def half_step(kind):
    """The most that one rounding to the type is off by, relative to the value."""
    return torch.finfo(TYPES[kind]).eps / 2


# ------------------------------------------------------------------------------ caches
def make_cache(kind, pages, page, kv, dim, layout="token", fill=float("nan")):
    """Keys and values of [pages][page][kv][dim] by index, in one of several orders in memory."""
    t = TYPES[kind]
    if layout == "token":       # [pages][page][kv][dim] each
        keys, values = (torch.full((pages, page, kv, dim), fill, dtype=t, device="cuda") for _ in range(2))
    elif layout == "head":      # [pages][kv][page][dim]
        keys, values = (torch.full((pages, kv, page, dim), fill, dtype=t, device="cuda").transpose(1, 2) for _ in range(2))
    elif layout == "joined":    # [pages][2][page][kv][dim]
        both = torch.full((pages, 2, page, kv, dim), fill, dtype=t, device="cuda")
        keys, values = both[:, 0], both[:, 1]
    else:                       # rows of a token padded by 8 elements
        assert layout == "padded"
        keys, values = (torch.full((pages, page, kv * dim + 8), fill, dtype=t, device="cuda")[..., :kv * dim]
                        .unflatten(-1, (kv, dim)) for _ in range(2))
    return keys, values


def describe(keys, values, kind):
    assert keys.stride() == values.stride() and keys.stride(3) == 1
    return native.PagedCache(keys=keys.data_ptr(), values=values.data_ptr(), page_stride=keys.stride(0),
                             slot_stride=keys.stride(1), head_stride=keys.stride(2), pages=keys.shape[0],
                             page_size=keys.shape[1], kv_heads=keys.shape[2], head_dim=keys.shape[3],
                             type=native.TYPES[kind])


def make_tables(rng, lengths, page, pages, width):
    """Tables of pages in random order, -1 behind what the lengths need."""
    held = [-(-n // page) for n in lengths]
    order = rng.permutation(pages)[:sum(held)]
    tables = np.full((len(lengths), width), -1, np.int32)
    at = 0
    for r, h in enumerate(held):
        tables[r, :h] = order[at:at + h]
        at += h
    return tables


# ------------------------------------------------------------------------------ attention
def attend(cache, q, heads, tables, lengths, out, lse=None, scale=None, window=0, workspace=None):
    dim, rows = cache.head_dim, tables.shape[0]
    size = lib().plamo_kernel_attention_paged_workspace(rows, heads, cache.kv_heads, dim)
    if workspace is None:
        # of arbitrary contents: the call reads nothing that it has not written
        workspace = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
    native.call(lib().plamo_kernel_attention_paged, cache, q.data_ptr(), q.stride(0), heads, tables.data_ptr(),
                tables.shape[1], lengths.data_ptr(), rows, 1 / math.sqrt(dim) if scale is None else scale, window,
                out.data_ptr(), out.stride(0), 0 if lse is None else lse.data_ptr(), workspace.data_ptr(),
                workspace.numel(), stream())
    return workspace


def attend64(keys, values, q, tables, lengths, scale, window=0):
    """-> out [rows][heads * dim], lse [rows][heads], and how far a kernel with FP32 sums may be off
    them before its last rounding (for both)."""
    pages, page, kv, dim = keys.shape
    rows, heads = q.shape[0], q.shape[1] // dim
    out, lse, slack, lse_slack = [], [], [], []
    for r in range(rows):
        n = min(max(int(lengths[r]), 0), tables.shape[1] * page)
        first = max(0, n - window) if window else 0
        at = [j for j in range(first, n) if 0 <= tables[r][j // page] < pages]
        o = torch.zeros(heads, dim, dtype=torch.float64)
        e = torch.full((heads,), -math.inf, dtype=torch.float64)
        s_o, s_e = torch.zeros(heads, dim, dtype=torch.float64), torch.zeros(heads, dtype=torch.float64)
        if at:
            where = torch.tensor([int(tables[r][j // page]) for j in at]), torch.tensor([j % page for j in at])
            k, v = (c[where[0].to(c.device), where[1].to(c.device)].double().cpu() for c in (keys, values))
            x = q[r].double().cpu().view(heads, dim)
            for h in range(heads):
                g = h // (heads // kv)
                score = (k[:, g] @ x[h]) * scale
                e[h] = torch.logsumexp(score, 0)
                share = torch.exp(score - e[h])
                o[h] = share @ v[:, g]
                # a score is a sum of `dim` products in FP32, scaled (2^-23 each: the sum may be
                # truncated); the exponential and its argument add 2^-21 of the largest score and of 1
                most = (k[:, g].abs() @ x[h].abs()).max() * abs(scale)
                s_e[h] = float(most) * (dim + 4) * 2.0 ** -23 + 2.0 ** -21 * (1 + float(score.abs().max()))
                # weights are off by twice that (numerator and sum) and by two halves' rounding, 2^-16;
                # sums over the keys are chains of a quarter of the keys' tiles and of the joins
                s_o[h] = (share @ v[:, g].abs()) * (2 * float(s_e[h]) + 2.0 ** -16 + (len(at) / 128 + 64) * 2.0 ** -23)
                s_e[h] += 2.0 ** -22 * abs(float(e[h])) + 2.0 ** -20
        out.append(o.reshape(-1))
        lse.append(e)
        slack.append(s_o.reshape(-1))
        lse_slack.append(s_e)
    return torch.stack(out), torch.stack(lse), torch.stack(slack), torch.stack(lse_slack)


# ------------------------------------------------------------------------------ projection rows
def paged_qkv(cache, kind, qkv, heads, slots, q, positions=None, q_norm=None, k_norm=None, rope=None):
    source = {v: k for k, v in TYPES.items()}[qkv.dtype]
    at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    native.call(lib().plamo_kernel_paged_qkv, cache, qkv.data_ptr(), native.TYPES[source], qkv.stride(0), heads, at(q_norm),
                at(k_norm), at(rope), 0 if rope is None else rope.shape[0], at(positions), slots.data_ptr(), qkv.shape[0],
                q.data_ptr(), q.stride(0), stream())


def rope_words(rows, half, base=10000.0):
    """[rows][half] BF16 cos | sin << 16, and the two as they are read, in 64 bits."""
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * base ** (-torch.arange(half, dtype=torch.float64) / half)
    cos, sin = torch.cos(angle).to(torch.bfloat16), torch.sin(angle).to(torch.bfloat16)
    word = lambda t: t.view(torch.int16).to(torch.int32) & 0xFFFF  # noqa: E731
    return (word(cos) | (word(sin) << 16)).to(torch.int32), cos.double(), sin.double()


def qkv64(qkv, heads, kv, dim, positions, cos, sin, gains):
    """-> rows [tokens][heads + 2 kv][dim] as they are to be written, before rounding, and a bound of
    what FP32 arithmetic may be off them."""
    x = qkv.double().cpu().view(qkv.shape[0], heads + 2 * kv, dim).clone()
    turned = slice(0, heads + kv)
    if gains is not None:
        g = 1 + torch.cat([gains[0].double().cpu().expand(heads, dim), gains[1].double().cpu().expand(kv, dim)])
        x[:, turned] = x[:, turned] / torch.sqrt((x[:, turned] ** 2).mean(-1, keepdim=True) + 1e-6) * g
    size = x.abs()
    if cos is not None:
        at = positions.long().cpu().clamp(0, cos.shape[0] - 1)
        c, s = cos[at][:, None], sin[at][:, None]
        a, b = x[:, turned, :dim // 2].clone(), x[:, turned, dim // 2:].clone()
        x[:, turned, :dim // 2], x[:, turned, dim // 2:] = a * c - b * s, b * c + a * s
        both = a.abs() + b.abs()
        size[:, turned, :dim // 2], size[:, turned, dim // 2:] = both, both
    # the sum of squares is off by 40 roundings at most (16 in a lane, 4 joins, twice for a product), half
    # of which reach its root; a dozen more follow
    return x, size * 32 * 2.0 ** -24


# ------------------------------------------------------------------------------ tables
def tables_step(lengths, counts, tables, free, page, pages, capacity):
    """One request after the other, on lists (changed in place) -> offsets, slots, positions, status.
    Nothing changes with a status other than 0."""
    width = len(tables[0])
    status, back, take = 0, 0, 0
    for length, count in zip(lengths, counts):
        if length < 0 or count < -1:
            status |= 8
            continue
        held, after = -(-length // page), 0 if count < 0 else -(-(length + count) // page)
        if max(held, after) > width:
            status |= 2
        if count < 0:
            back += held
        else:
            take += after - held
    if len(free) + back > pages:
        status |= 8
    elif take > len(free) + back:
        status |= 1
    if sum(c for n, c in zip(lengths, counts) if c > 0 and n >= 0) > capacity:
        status |= 4
    if status:
        return [0] * (len(lengths) + 1), [-1] * capacity, [-1] * capacity, status
    offsets, slots, positions = [0], [], []
    for r, count in enumerate(counts):
        if count < 0:
            free.extend(tables[r][:-(-lengths[r] // page)])
            lengths[r] = 0
    for r, count in enumerate(counts):
        for _ in range(max(count, 0)):
            n = lengths[r]
            if n % page == 0:
                tables[r][n // page] = free.pop()
            slots.append(tables[r][n // page] * page + n % page)
            positions.append(n)
            lengths[r] += 1
        offsets.append(len(slots))
    pad = [-1] * (capacity - len(slots))
    return offsets, slots + pad, positions + pad, 0


# ------------------------------------------------------------------------------ sampling
def sample(logits, n, uniform, temperature=None, top_k=None, top_p=None, min_p=None, prob=True, workspace=None):
    kind = {v: k for k, v in TYPES.items()}[logits.dtype]
    rows = logits.shape[0]
    token = torch.full((rows + 1,), -7, dtype=torch.int32, device="cuda")
    share = torch.full((rows + 1,), -7.0, device="cuda") if prob else None
    size = lib().plamo_kernel_sample_workspace(rows, n)
    if workspace is None:
        workspace = torch.full((max(16, size),), 0xFF, dtype=torch.uint8, device="cuda")
    at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    native.call(lib().plamo_kernel_sample, logits.data_ptr(), native.TYPES[kind], logits.stride(0), n, rows, at(temperature),
                at(top_k), at(top_p), at(min_p), uniform.data_ptr(), token.data_ptr(), at(share), workspace.data_ptr(),
                workspace.numel(), stream())
    return token, share


def sample64(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row (64-bit values) -> token, probability."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    if not np.any(x > -np.inf):
        return -1, 0.0
    if not temperature > 0:
        return int(np.argmax(x)), 1.0
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    top = x[order[0]]
    w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / temperature)) if np.isfinite(top) else \
        (x[order] == top).astype(np.float64)
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        keep = before < top_p * w.sum()
        keep[0] = True
        order, w = order[keep], w[keep]
    if min_p > 0:
        keep = w >= min(min_p, 1.0)
        order, w = order[keep], w[keep]
    sums = np.cumsum(w)
    at = min(int(np.searchsorted(sums, u * sums[-1], side="right")), int(np.flatnonzero(w)[-1]))
    return int(order[at]), float(w[at] / sums[-1])
