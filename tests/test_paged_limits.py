"""Sizes next to the 32-bit numbers that the paged kernels count in: refused before any device work (no GPU is needed,
the addresses here are never read)."""
import pytest

from test_paged_refusals import cache, call


@pytest.mark.parametrize("changed", [dict(rows=(1 << 30) + 1), dict(rows=2 ** 31 - 1), dict(capacity=(1 << 30) + 1),
                                     dict(capacity=2 ** 31 - 1)])
def test_rows_and_places_of_tables(changed):
    rc, message = call("plamo_kernel_paged_tables", **changed)
    assert rc == 1 and message.startswith("paged tables: ")
