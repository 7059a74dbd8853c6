"""Calls that the paged and sampling entry points refuse: PLAMO_EINVAL and a message, before any device work
(no GPU is needed: the addresses here are never read)."""
import ctypes
import math

import pytest

from plamo_hip import native

A = 1 << 20  # an aligned address


def call(name, **changed):
    spec = dict(CALLS[name])
    assert set(changed) <= set(spec)
    spec.update(changed)
    err = ctypes.create_string_buffer(256)
    rc = getattr(native.load(), name)(*spec.values(), err, 256)
    return rc, err.value.decode()


def cache(**changed):
    spec = dict(keys=A, values=A, page_stride=16 * 128, slot_stride=128, head_stride=128, pages=10, page_size=16, kv_heads=1,
                head_dim=128, type=0)
    spec.update(changed)
    return native.PagedCache(**spec)


CALLS = {
    "plamo_kernel_paged_tables": dict(lengths=A, counts=A, rows=3, tables=A, width=4, page_size=16, free_pages=A,
                                      free_count=A, pages=10, lengths_out=A, free_out=A, offsets=A, slots=A, positions=A,
                                      capacity=5, status=A, stream=0),
    "plamo_kernel_paged_qkv": dict(cache=cache(), qkv=A, type=2, qkv_stride=18 * 128, heads=16, q_norm=A, k_norm=A, rope=A,
                                   rope_rows=100, positions=A, slots=A, tokens=4, q=A, q_stride=2048, stream=0),
    "plamo_kernel_attention_paged": dict(cache=cache(), q=A, q_stride=2048, heads=16, tables=A, width=4, lengths=A, rows=3,
                                         scale=0.1, window=0, out=A, out_stride=2048, lse=A, workspace=A,
                                         workspace_bytes=1 << 40, stream=0),
    "plamo_kernel_sample": dict(logits=A, type=0, stride=1000, n=1000, rows=3, temperature=A, top_k=A, top_p=A, min_p=A,
                                uniform=A, token=A, prob=A, workspace=A, workspace_bytes=1 << 40, stream=0),
}


@pytest.mark.parametrize("changed", [
    dict(rows=0), dict(rows=-1), dict(width=0), dict(page_size=0), dict(pages=0), dict(capacity=-1),
    dict(pages=1 << 20, page_size=1 << 12), dict(lengths=0), dict(counts=0), dict(tables=0), dict(free_pages=0),
    dict(free_count=0), dict(lengths_out=0), dict(free_out=0), dict(offsets=0), dict(slots=0), dict(positions=0),
    dict(status=0)])
def test_tables(changed):
    rc, message = call("plamo_kernel_paged_tables", **changed)
    assert rc == 1 and message.startswith("paged tables: ")


CACHES = [dict(type=2), dict(type=-1), dict(head_dim=96), dict(head_dim=0), dict(kv_heads=0), dict(kv_heads=257),
          dict(pages=0), dict(page_size=0), dict(pages=1 << 20, page_size=1 << 12), dict(keys=0), dict(values=0),
          dict(keys=A + 8), dict(values=A + 2), dict(page_stride=4), dict(slot_stride=130), dict(head_stride=-8),
          dict(page_stride=-2048), dict(slot_stride=-128), dict(slot_stride=(1 << 24) + 8), dict(page_stride=1 << 41)]


@pytest.mark.parametrize("changed", CACHES)
@pytest.mark.parametrize("name", ["plamo_kernel_paged_qkv", "plamo_kernel_attention_paged"])
def test_caches(name, changed):
    rc, message = call(name, cache=cache(**changed))
    assert rc == 1 and message.startswith("paged cache: ")


def test_no_cache():
    for name in ("plamo_kernel_paged_qkv", "plamo_kernel_attention_paged"):
        assert call(name, cache=None) == (1, "null paged cache")


@pytest.mark.parametrize("changed", [
    dict(type=1), dict(type=3), dict(heads=0), dict(heads=4097), dict(cache=cache(kv_heads=3)), dict(tokens=-1),
    dict(qkv_stride=18 * 128 - 4), dict(qkv_stride=18 * 128 + 1), dict(type=0, qkv_stride=18 * 128 + 4), dict(q_stride=2040),
    dict(q_stride=2050), dict(tokens=1 << 30), dict(qkv=0), dict(q=0), dict(slots=0), dict(qkv=A + 4), dict(q=A + 8),
    dict(q_norm=A + 2), dict(k_norm=A + 8), dict(rope=A + 8), dict(positions=0), dict(rope_rows=0)])
def test_qkv(changed):
    rc, message = call("plamo_kernel_paged_qkv", **changed)
    assert rc == 1 and message.startswith("paged qkv: ")


@pytest.mark.parametrize("changed", [
    dict(heads=0), dict(heads=4097), dict(cache=cache(kv_heads=3)), dict(rows=0), dict(rows=(1 << 20) + 1), dict(width=0),
    dict(width=1 << 27), dict(window=-1), dict(scale=math.nan), dict(scale=math.inf), dict(q_stride=2040), dict(q_stride=2052),
    dict(out_stride=1024), dict(out_stride=2049), dict(q=0), dict(out=0), dict(tables=0), dict(lengths=0), dict(q=A + 2),
    dict(out=A + 8), dict(workspace=0), dict(workspace=A + 8), dict(workspace_bytes=1000)])
def test_attention(changed):
    rc, message = call("plamo_kernel_attention_paged", **changed)
    assert rc == 1 and message.startswith("paged attention: ")


@pytest.mark.parametrize("changed", [
    dict(type=3), dict(type=-1), dict(n=0), dict(n=(1 << 20) + 1), dict(rows=0), dict(rows=(1 << 20) + 1), dict(stride=999),
    dict(stride=-1000), dict(logits=0), dict(uniform=0), dict(token=0), dict(logits=A + 1), dict(type=2, logits=A + 2),
    dict(workspace_bytes=-1)])
def test_sample(changed):
    rc, message = call("plamo_kernel_sample", **changed)
    assert rc == 1 and message.startswith("sample: ")


def test_workspace_sizes():
    lib = native.load()
    for bad in ((0, 16, 1, 128), (1, 0, 1, 128), (1, 16, 3, 128), (1, 4097, 1, 64), (1, 16, 0, 128), (1, 16, 1, 0)):
        assert lib.plamo_kernel_attention_paged_workspace(*bad) == -1
    one = lib.plamo_kernel_attention_paged_workspace(1, 16, 1, 128)
    assert 0 < one < lib.plamo_kernel_attention_paged_workspace(1000, 16, 1, 128) < 1 << 30
    exact = dict(workspace_bytes=lib.plamo_kernel_attention_paged_workspace(3, 16, 1, 128) - 1)
    assert call("plamo_kernel_attention_paged", **exact)[0] == 1
    for bad in ((0, 100), (1, 0), (1, (1 << 20) + 1)):
        assert lib.plamo_kernel_sample_workspace(*bad) == -1
    assert lib.plamo_kernel_sample_workspace(4, 107520) >= 0
