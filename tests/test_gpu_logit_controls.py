"""Penalties, n-grams, biases and masks on rows of logits, against 64 bits."""
import math

import numpy as np
import pytest
import torch

from paged_common import TYPES, half_step
from speculate_common import controls, controls64, lines_of, put, random_parents

pytestmark = pytest.mark.gpu


def check(logits, n, spec, sequences, out_kind=None, rows_of=None, pad=0, in_place=False):
    """`spec`: host values by the fields' names, `said` and `ngram` among them."""
    rows = logits.shape[0]
    kind = {v: k for k, v in TYPES.items()}[logits.dtype]
    out_kind = out_kind or kind
    float_names = ("repetition", "presence", "frequency", "bias")
    device = {k: put(v, torch.float32 if k in float_names else torch.int32) for k, v in spec.items() if k != "paths"}
    if in_place:
        out, before = logits, logits.clone()
    else:
        out, before = torch.full((rows, n + pad), 7.0, dtype=TYPES[out_kind], device="cuda")[:, :n], logits
    x = before[:, :n].double().cpu().numpy()
    controls(logits, n, out, device, sequences)
    torch.cuda.synchronize()
    got = out[:, :n].double().cpu().numpy()
    masks = np.array(spec["masks"], dtype=np.int64).astype(np.uint32).view(np.uint8) if "masks" in spec else None
    for t in range(rows):
        r = t if rows_of is None else rows_of[t]
        if r < 0:
            assert np.array_equal(got[t], x[t] if in_place else np.full(n, 7.0)), t
            continue
        said = []
        if "history" in spec:
            said = list(np.array(spec["history"])[r][:max(0, min(spec["history_lengths"][r], len(spec["history"][r])))])
        said = [int(s) for s in said] + (spec["paths"][t] if "paths" in spec else [])
        one = {k: float(np.float32(spec[k][r])) for k in ("repetition", "presence", "frequency") if k in spec}
        bias = list(zip(spec["bias_ids"][r], np.float32(spec["bias"][r]).astype(float))) if "bias_ids" in spec else []
        mask = None
        if masks is not None:
            m = spec["mask_rows"][t] if "mask_rows" in spec else t
            if 0 <= m < len(masks):
                mask = np.unpackbits(masks[m], bitorder="little")[:n].astype(bool)
        want, slack = controls64(x[t], said, ngram=spec["ngram"][r] if "ngram" in spec else 0, bias=bias, mask=mask, **one)
        fine = np.isfinite(want)
        assert np.array_equal(fine, np.isfinite(got[t])) and np.array_equal(got[t][~fine], want[~fine], equal_nan=True), t
        off = np.abs(got[t][fine] - want[fine]) - slack[fine] - np.abs(want[fine]) * half_step(out_kind) - 2.0 ** -24
        assert np.all(off <= 0), (t, off.max())
        plain = np.setdiff1d(np.arange(n), [s for s in said] + [b for b, _ in bias])
        plain = plain[fine[plain]]
        assert np.array_equal(got[t][plain], x[t][plain]), t  # what nothing says keeps its bits
    return out


def logits_of(kind, rows, n, seed=0, stride=None):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(rows, stride or n, generator=g, device="cuda") * 3).to(TYPES[kind])


def history_of(rng, rows, width, n, few=12):
    words = rng.integers(0, n, few)
    return words[rng.integers(0, few, (rows, width))].tolist(), rng.integers(width // 2, width + 1, rows).tolist()


def masks_of(rng, count, n, part=0.5):
    words = -(-n // 32)
    bits = rng.random((count, words * 32)) < part
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32).view(np.int32).tolist()


@pytest.mark.parametrize("n", [1, 7, 8, 33, 4095, 4096, 4097, 5003, 20000])
@pytest.mark.parametrize("kind,out_kind", [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32"), ("fp32", "fp32")])
def test_everything_at_once(kind, out_kind, n):
    rng, rows = np.random.default_rng(n), 4
    history, lengths = history_of(rng, rows, 60, n)
    ids = np.stack([rng.permutation(max(n, 9))[:9] for _ in range(rows)])
    spec = dict(history=history, history_lengths=lengths, repetition=[1.3, 1.0, 0.8, 1.1], presence=[0.5, 0, -0.2, 0.1],
                frequency=[0.2, 0.1, 0, -0.3], ngram=[2, 3, 0, 1], bias_ids=ids.tolist(), bias=rng.standard_normal((rows, 9)).tolist(),
                masks=masks_of(rng, 3, n), mask_rows=[2, -1, 0, 7])
    for pad in (0, 1, 5):
        check(logits_of(kind, rows, n, n, n + pad), n, spec, rows, out_kind, pad=pad)
    if kind == out_kind:
        check(logits_of(kind, rows, n, n, n + 3), n, spec, rows, out_kind, in_place=True)


@pytest.mark.parametrize("one", ["repetition", "presence", "frequency"])
def test_one_penalty(one):
    rng, n = np.random.default_rng(1), 500
    history, lengths = history_of(rng, 3, 40, n)
    check(logits_of("fp32", 3, n), n, {"history": history, "history_lengths": lengths, one: [1.5, 0.3, 0.7]}, 3)


@pytest.mark.parametrize("repetition,presence,frequency", [(0.0, 0.5, 0.5), (-2.0, 0.0, 0.1), (math.nan, math.nan, math.nan),
                                                           (1.0, math.nan, 0.25), (1.2, 0.0, math.nan)])
def test_controls_that_are_off(repetition, presence, frequency):
    rng, n = np.random.default_rng(2), 300
    history, lengths = history_of(rng, 2, 50, n)
    check(logits_of("bf16", 2, n), n, dict(history=history, history_lengths=lengths, repetition=[repetition] * 2,
                                           presence=[presence] * 2, frequency=[frequency] * 2), 2)


@pytest.mark.parametrize("ngram", [-1, 0, 1, 2, 3, 4, 9, 50, 51, 2 ** 31 - 1])
def test_ngrams(ngram):
    rng, n = np.random.default_rng(3), 100
    history = rng.integers(0, 3, (4, 50))
    history[3, 25:] = history[3, :25]  # repeats a long one
    check(logits_of("fp32", 4, n), n, dict(history=history.tolist(), history_lengths=[50, 1, 7, 50], ngram=[ngram] * 4), 4)


def test_histories():
    """Lengths below zero and past the width, tokens outside the vocabulary, a stride past the width."""
    n = 64
    history = [[5, -3, 64, 5, 2 ** 31 - 1, 6], [7] * 6, [8] * 6, [9] * 6]
    spec = dict(history=history, history_lengths=[6, -5, 0, 100], repetition=[2.0] * 4, frequency=[0.5] * 4, ngram=[2] * 4)
    check(logits_of("fp32", 4, n), n, spec, 4)


def test_a_long_history():
    rng, n = np.random.default_rng(4), 5000
    width = 1 << 17
    history = rng.integers(0, 50, (2, width))
    history[1] = 3  # one token 131,072 times
    check(logits_of("fp32", 2, n), n, dict(history=history.tolist(), history_lengths=[width, width], frequency=[1e-3, 2.0 ** -10],
                                           repetition=[1.2, 1.0]), 2)


def test_biases():
    """The last of equal ids counts; ids outside the vocabulary are skipped; infinities."""
    n = 100
    ids = [[5, 6, 5, -1, 100, 7, 5], [99, 0, 0, 1, 2, 2 ** 31 - 1, 3]]
    bias = [[1.0, math.inf, 2.0, 9.0, 9.0, -math.inf, 4.0], [0.5, 1.0, -1.0, math.nan, 0.0, 8.0, -2.0]]
    check(logits_of("fp32", 2, n), n, dict(bias_ids=ids, bias=bias), 2)
    rng = np.random.default_rng(5)
    ids = rng.integers(-1, 6000, (2, 4096))
    check(logits_of("bf16", 2, 5000), 5000, dict(bias_ids=ids.tolist(), bias=rng.standard_normal((2, 4096)).tolist()), 2)


def test_masks():
    rng, n = np.random.default_rng(6), 131
    none = [0] * 5
    check(logits_of("bf16", 3, n), n, dict(masks=masks_of(rng, 3, n)), 3)
    out = check(logits_of("bf16", 2, n), n, dict(masks=[none, [-1] * 5], mask_rows=[0, 1]), 2)
    assert torch.all(out[0] == -math.inf) and torch.isfinite(out[1]).all()
    check(logits_of("fp16", 2, n), n, dict(masks=[none, [-1] * 5], mask_rows=[-2 ** 31, 2]), 2)


def test_odd_logits():
    """Infinities and NaN stay what arithmetic makes of them; what is banned is minus infinity whatever it was."""
    x = logits_of("fp32", 2, 40)
    x[:, 3], x[:, 4], x[:, 5], x[:, 6], x[:, 7], x[:, 8] = math.inf, -math.inf, math.nan, math.nan, 0.0, -0.0
    spec = dict(history=[[3, 4, 5, 7, 8, 9]] * 2, history_lengths=[6, 6], repetition=[1.5, 1.0], presence=[0.5, 0.25],
                masks=[[~(1 << 6), -1]], mask_rows=[0, -1])
    check(x, 40, spec, 2)


def test_nothing_on():
    x = logits_of("bf16", 3, 5001)
    out = check(x, 5001, {}, 3)
    assert torch.equal(out.view(torch.int16), x.view(torch.int16))


@pytest.mark.parametrize("counts", [[3, 1, 7], [0, 5, 0, 2], [40, 70], [1] * 70 + [3] * 70])
def test_trees(counts):
    """Each node's row has the path to it behind the history; rows behind the last request are left."""
    rng, n = np.random.default_rng(len(counts)), 700
    offsets = np.concatenate([[0], np.cumsum(counts)]).tolist()
    total, rows = offsets[-1], offsets[-1] + 2
    words = -(-max(counts) // 32)
    tokens = rng.integers(0, 5, rows)
    bits, paths, rows_of = np.zeros((rows, words), np.uint32), [], []
    for r, c in enumerate(counts):
        for line in lines_of(random_parents(rng, c)):
            for j in line:
                bits[len(paths), j // 32] |= np.uint32(1 << (j % 32))
            paths.append([int(tokens[offsets[r] + j]) for j in line])
            rows_of.append(r)
    sequences = len(counts)
    spec = dict(history=rng.integers(0, 5, (sequences, 9)).tolist(), history_lengths=rng.integers(0, 10, sequences).tolist(),
                offsets=offsets, tokens=tokens.tolist(), ancestors=bits.view(np.int32).tolist(), ngram=[3] * sequences,
                repetition=rng.uniform(0.7, 1.4, sequences).tolist(), frequency=rng.uniform(0, 0.5, sequences).tolist(),
                masks=masks_of(rng, 4, n, 0.9), mask_rows=rng.integers(-1, 4, rows).tolist(), paths=paths + [[], []])
    check(logits_of("bf16", rows, n), n, spec, sequences, "fp32", rows_of + [-1, -1])
    check(logits_of("bf16", rows, n), n, spec, sequences, rows_of=rows_of + [-1, -1], in_place=True)
    del spec["ancestors"], spec["tokens"], spec["paths"]  # the histories alone
    check(logits_of("fp32", rows, n), n, spec, sequences, rows_of=rows_of + [-1, -1])
    del spec["history"], spec["history_lengths"]
    assert total == len(rows_of)
    check(logits_of("fp16", rows, n), n, spec, sequences, rows_of=rows_of + [-1, -1])


def test_paths_without_a_history():
    n = 50
    spec = dict(offsets=[0, 3], tokens=[4, 5, 6], ancestors=[[1], [3], [5]], frequency=[0.5], paths=[[4], [4, 5], [4, 6]])
    check(logits_of("fp32", 3, n), n, spec, 1, rows_of=[0, 0, 0])
