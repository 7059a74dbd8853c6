"""Sizes next to the 32-bit numbers that the paged kernels count in: refused before any device work (no GPU is needed,
the addresses here are never read)."""
import pytest

from test_paged_refusals import cache, call


@pytest.mark.parametrize("changed", [dict(rows=(1 << 30) + 1), dict(rows=2 ** 31 - 1), dict(capacity=(1 << 30) + 1),
                                     dict(capacity=2 ** 31 - 1)])
def test_rows_and_places_of_tables(changed):
    rc, message = call("plamo_kernel_paged_tables", **changed)
    assert rc == 1 and message.startswith("paged tables: ")


@pytest.mark.parametrize("rows,heads,kv,window", [(1 << 20, 256, 1, 1), (1 << 20, 4096, 1, 1), (1 << 16, 4096, 1, 1),
                                                  (1 << 20, 512, 2, 0)])
def test_workgroups_of_attention(rows, heads, kv, window):
    """More threads along the grid than a launch has."""
    rc, message = call("plamo_kernel_attention_paged", cache=cache(kv_heads=kv), q_stride=heads * 128, heads=heads, rows=rows,
                       width=1000, window=window, out_stride=heads * 128, workspace_bytes=1 << 60)
    assert rc == 1 and message.startswith("paged attention: too many rows")
