"""Calls that the entry points of a speculative step refuse: PLAMO_EINVAL and a message, before any device work (no GPU is
needed: the addresses here are never read)."""
import ctypes
import math

import pytest

from plamo_hip import native
from test_paged_refusals import A, CACHES, cache


def controls(**changed):
    spec = dict(history=A, history_lengths=A, offsets=A, tokens=A, ancestors=A, repetition=A, presence=A, frequency=A, ngram=A,
                bias_ids=A, bias=A, masks=A, mask_rows=A, history_stride=100, mask_stride=40, sequences=2, history_width=100,
                words=1, bias_width=5, mask_count=3)
    spec.update(changed)
    return native.LogitControls(**spec)


def call(name, **changed):
    spec = dict(CALLS[name])
    assert set(changed) <= set(spec)
    spec.update(changed)
    err = ctypes.create_string_buffer(256)
    rc = getattr(native.load(), name)(*spec.values(), err, 256)
    return rc, err.value.decode()


CALLS = {
    "plamo_kernel_paged_tree": dict(lengths=A, offsets=A, rows=3, parents=A, tokens=10, window=0, positions=A, ancestors=A,
                                    words=1, stream=0),
    "plamo_kernel_attention_paged_tree": dict(cache=cache(), q=A, q_stride=2048, heads=16, tables=A, width=4, lengths=A,
                                              offsets=A, rows=3, tokens=10, positions=A, ancestors=A, words=1, scale=0.1,
                                              window=0, out=A, out_stride=2048, lse=A, workspace=A, workspace_bytes=1 << 40,
                                              stream=0),
    "plamo_kernel_logit_controls": dict(controls=controls(), logits=A, type=0, stride=1000, n=1000, rows=3, out=2 * A, out_type=0,
                                        out_stride=1000, stream=0),
    "plamo_kernel_paged_accept": dict(lengths=A, offsets=A, rows=3, parents=A, tokens=A, drawn=A, capacity=10, given=A, tables=A,
                                      width=4, page_size=16, free_pages=A, free_count=A, pages=10, lengths_out=A, free_out=A,
                                      accepted=A, accepted_counts=A, last=A, nodes=5, source=A, target=A, status=A, stream=0),
    "plamo_kernel_paged_move": dict(caches=cache(), layers=1, source=A, target=A, groups=3, group=5, stream=0),
}


@pytest.mark.parametrize("changed", [
    dict(rows=0), dict(rows=(1 << 20) + 1), dict(tokens=-1), dict(tokens=(1 << 24) + 1), dict(words=0), dict(words=33),
    dict(window=-1), dict(lengths=0), dict(offsets=0), dict(parents=0), dict(positions=0), dict(ancestors=0)])
def test_tree(changed):
    rc, message = call("plamo_kernel_paged_tree", **changed)
    assert rc == 1 and message.startswith("paged tree: ")


@pytest.mark.parametrize("changed", [
    dict(heads=0), dict(heads=4097), dict(cache=cache(kv_heads=3)), dict(rows=0), dict(rows=(1 << 20) + 1), dict(width=0),
    dict(width=1 << 27), dict(tokens=-1), dict(tokens=(1 << 20) + 1), dict(tokens=1 << 20, heads=2048, q_stride=1 << 20, out_stride=1 << 20),
    dict(window=-1), dict(scale=math.nan), dict(scale=-math.inf), dict(q_stride=2040), dict(q_stride=2052), dict(out_stride=1024),
    dict(out_stride=2049), dict(q=0), dict(out=0), dict(tables=0), dict(lengths=0), dict(offsets=0), dict(q=A + 2), dict(out=A + 8),
    dict(positions=0), dict(words=0), dict(words=33), dict(workspace=0), dict(workspace=A + 8), dict(workspace_bytes=1000)])
def test_attention(changed):
    rc, message = call("plamo_kernel_attention_paged_tree", **changed)
    assert rc == 1 and message.startswith("tree attention: ")


@pytest.mark.parametrize("changed", CACHES)
@pytest.mark.parametrize("name", ["plamo_kernel_attention_paged_tree", "plamo_kernel_paged_move"])
def test_caches(name, changed):
    field = "cache" if "attention" in name else "caches"
    rc, message = call(name, **{field: cache(**changed)})
    assert rc == 1 and message.startswith("paged cache: ")


def test_nothing_given():
    assert call("plamo_kernel_attention_paged_tree", cache=None) == (1, "null paged cache")
    assert call("plamo_kernel_paged_move", caches=None) == (1, "paged move: no caches")
    assert call("plamo_kernel_logit_controls", controls=None) == (1, "null logit controls")


@pytest.mark.parametrize("changed", [
    dict(type=3), dict(type=-1), dict(out_type=1), dict(type=2, out_type=0), dict(n=0), dict(n=(1 << 20) + 1), dict(rows=-1),
    dict(rows=(1 << 20) + 1), dict(n=1 << 20, rows=1 << 20, stride=1 << 20, out_stride=1 << 20), dict(stride=999), dict(out_stride=999),
    dict(stride=-1000), dict(logits=0), dict(out=0), dict(logits=A + 1), dict(out=2 * A + 1), dict(type=2, out_type=2, logits=A + 2),
    dict(out_type=2, out=2 * A + 2), dict(out=A, out_type=2), dict(out=A, out_stride=1001)] + [
        dict(controls=controls(**c)) for c in (
            dict(sequences=0), dict(sequences=(1 << 20) + 1), dict(offsets=0, ancestors=0, sequences=2), dict(history_lengths=0),
            dict(history_width=-1), dict(history_width=(1 << 17) + 1, history_stride=1 << 18), dict(history_stride=99), dict(offsets=0, sequences=3),
            dict(tokens=0), dict(words=0), dict(words=33), dict(bias=0), dict(bias_width=-1), dict(bias_width=4097),
            dict(mask_count=0), dict(mask_stride=31), dict(masks=A + 2), dict(mask_rows=0, mask_count=2))])
def test_controls(changed):
    rc, message = call("plamo_kernel_logit_controls", **changed)
    assert rc == 1 and message.startswith("logit controls: ")


@pytest.mark.parametrize("changed", [dict(rows=0), dict(rows=(1 << 20) + 1), dict(capacity=-1), dict(capacity=(1 << 24) + 1), dict(width=0),
                                     dict(nodes=-1), dict(nodes=(1 << 16) + 1), dict(page_size=0), dict(pages=0),
                                     dict(pages=1 << 20, page_size=1 << 12)] +
                         [{k: 0} for k in ("lengths", "offsets", "parents", "tokens", "drawn", "tables", "free_pages", "free_count",
                                           "lengths_out", "free_out", "accepted", "accepted_counts", "last", "source", "target", "status")])
def test_accept(changed):
    rc, message = call("plamo_kernel_paged_accept", **changed)
    assert rc == 1 and message.startswith("paged accept: ")


@pytest.mark.parametrize("changed", [dict(layers=0), dict(groups=-1), dict(group=0), dict(groups=1 << 30), dict(source=0), dict(target=0)])
def test_move(changed):
    rc, message = call("plamo_kernel_paged_move", **changed)
    assert rc == 1 and message.startswith("paged move: ")


@pytest.mark.parametrize("other", [dict(page_stride=32 * 128), dict(slot_stride=256), dict(head_stride=64), dict(pages=11), dict(page_size=8),
                                   dict(kv_heads=2), dict(head_dim=64), dict(type=1)])
def test_layers_that_differ(other):
    array = (native.PagedCache * 2)(cache(), cache(**other))
    rc, message = call("plamo_kernel_paged_move", caches=array, layers=2)
    assert rc == 1 and message == "paged move: caches must be alike but for their addresses"


def test_workspace_sizes():
    size = native.load().plamo_kernel_attention_paged_tree_workspace
    for bad in ((0, 10, 16, 1, 128), (1, -1, 16, 1, 128), (1, 10, 0, 1, 128), (1, 10, 16, 3, 128), (1, 10, 4097, 1, 64),
                (1, 10, 16, 0, 128), (1, 10, 16, 1, 0), ((1 << 20) + 1, 10, 16, 1, 128), (1, (1 << 20) + 1, 16, 1, 128)):
        assert size(*bad) == -1
    assert 0 < size(1, 1, 16, 1, 128) <= size(64, 2000, 16, 1, 128) < 1 << 30
    exact = dict(workspace_bytes=size(3, 10, 16, 1, 128) - 1)
    assert call("plamo_kernel_attention_paged_tree", **exact)[0] == 1
