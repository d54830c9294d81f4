"""What hidden keys hold, and outputs that lie where the queries do (GPU).

A key that a row does not see takes no part in it, whatever its K and V are: single tokens,
prompts whose items are cut into parts or not, tiles that come straight into LDS or through
registers. Tolerances as in test_gpu_attention.py.
"""
from __future__ import annotations

import pytest
import torch

from test_gpu_attention import BF16, F16, F32, FP8, make_pool, make_tables, queries_of, reference

pytestmark = pytest.mark.gpu

TYPES = [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8), (F32, F32), (F32, BF16)]
NAN, INF = float("nan"), float("inf")
VALUES = [(q, c, x) for q, c in TYPES for x in ([NAN] if c == FP8 else [NAN, INF, -INF])]


def poison(cache, slot, value):
    """``value`` in a row of a cache (NaN in 8 bits, which hold no infinities)."""
    rows = cache.float()
    rows[slot] = NAN if cache.dtype == FP8 else value
    cache.copy_(rows.to(cache.dtype))


def at_odd_address(t):
    flat = torch.zeros(t.numel() + 1, dtype=torch.float32, device="cuda").to(t.dtype)[1:]
    odd = flat.view(t.shape)
    odd.view(torch.uint8).copy_(t.view(torch.uint8))
    return odd


# Prompts of few items, which are cut into parts, and of enough items not to be.
@pytest.mark.parametrize("kv_heads, n", [(2, 1200), (2, 150), (16, 700)])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("query, cache, value", VALUES)
def test_rows_of_a_prompt_that_do_not_see_a_key(gpu, query, cache, value, which, kv_heads, n):
    """K or V of a key in the middle is no number: rows before it, and rows whose window has
    left it behind, do not show it, whether the caches are aligned or not."""
    from iekv.engine.attention import AttentionPlan, attend
    from iekv.engine.pools import KVPool

    bs, group, dim, window, sinks = 16, 4, 64, 90, 3
    key = n - 100
    blocks = -(-n // bs) + 1
    pool, k, v = make_pool(blocks, bs, kv_heads, dim, cache, 90)
    tables = make_tables([n], bs, blocks, 91)
    q = queries_of(n, kv_heads * group, dim, query, 92)
    want, tol = reference(q, k[0], v[0], bs, tables, [n], [n], window=window, sinks=sinks)
    poison({"k": k, "v": v}[which][0], tables[0][key // bs] * bs + key % bs, value)
    odd = KVPool([at_odd_address(k[0])], [at_odd_address(v[0])], bs)
    blind = [slice(0, key), slice(key + window, n)]
    for p in (pool, odd):
        plan = AttentionPlan(p, tables, [n], [n], kv_heads * group, window=window, sinks=sinks,
                             query_dtype=query)
        got = attend(plan, 0, q)
        for part in blind:
            assert ((got[part].double() - want[part]).abs() <= tol[part]).all()
        if which == "v" or value != value:          # K of infinities weighs as 0 or 1
            assert not torch.isfinite(got[key:key + window]).all(-1).any()
