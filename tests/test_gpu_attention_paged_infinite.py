"""Infinite values in pages (plamo_kernel_attention_paged): what is hidden reaches nothing; one that is seen makes its
dimension infinite or NaN, in the heads that see it, and no other."""
import math

import numpy as np
import pytest
import torch

from paged_common import TYPES, attend, attend64, describe, half_step, make_cache, make_tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 10), (256, 64)])
@pytest.mark.parametrize("n", [70, 1500])
def test_infinite_values(kind, dim, page, n):
    rng = np.random.default_rng([dim, page, n])
    lengths, heads, kv = [n, n], 4, 2
    tables = make_tables(rng, lengths, page, 2 * -(-n // page) + 1, -(-n // page))
    keys, values = make_cache(kind, 2 * -(-n // page) + 1, page, kv, dim, fill=math.inf)
    for r in range(2):
        for j in range(n):
            for cache in (keys, values):
                cache[int(tables[r, j // page]), j % page] = torch.from_numpy(rng.standard_normal((kv, dim)))
    q = torch.from_numpy(rng.standard_normal((2, heads * dim))).to(TYPES[kind]).cuda()
    device, size = torch.from_numpy(tables).cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    plain, out = (torch.zeros(2, heads * dim, dtype=TYPES[kind], device="cuda") for _ in range(2))
    attend(describe(keys, values, kind), q, heads, device, size, plain)
    want, _, slack, _ = attend64(keys, values, q, tables, lengths, 1 / math.sqrt(dim))
    assert torch.all((plain.double().cpu() - want).abs() <= want.abs() * half_step(kind) + slack * (1 + half_step(kind)) + 1e-7)
    at = n - 3
    values[int(tables[0, at // page]), at % page, 1, 5] = -math.inf
    attend(describe(keys, values, kind), q, heads, device, size, out)
    out, plain = out.view(2, heads, dim), plain.view(2, heads, dim)
    touched = torch.zeros_like(out, dtype=torch.bool)
    touched[0, 2:, 5] = True
    assert not torch.isfinite(out[touched]).any()
    assert torch.equal(out[~touched], plain[~touched])
