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


STEPS = {
    "tokens": ([37, 500, 64, 1], [1, 1, 1, 1], 0),
    "two tokens": ([300, 77], [2, 2], 0),
    "long": ([5001, 4000], [1, 2], 0),
    "prompts": ([333, 200], [333, 70], 0),
    "prefix": ([2100 + i for i in range(40)], [1] * 40, 128),
}


@pytest.mark.parametrize("step", list(STEPS))
@pytest.mark.parametrize("hidden", [False, True])
@pytest.mark.parametrize("query, cache", [(BF16, BF16), (F16, FP8), (F32, F32)])
def test_outputs_in_place_of_the_queries(gpu, query, cache, hidden, step):
    """The same bits as into a tensor of its own, also where hidden keys that are no numbers
    make rows be done again."""
    from iekv.engine.attention import AttentionPlan, attend

    contexts, queries, shared = STEPS[step]
    bs, kv_heads, group, dim = 16, 4, 2, 64
    blocks = shared + sum(-(-c // bs) for c in contexts) + 2
    pool, k, v = make_pool(blocks, bs, kv_heads, dim, cache, 93)
    tables = make_tables(contexts, bs, blocks, 94, shared)
    if hidden:
        for table, n, m in zip(tables, contexts, queries):
            if m > 1:
                poison(v[0], table[(n - 1) // bs] * bs + (n - 1) % bs, INF)
    q = queries_of(sum(queries), kv_heads * group, dim, query, 95)
    plan = AttentionPlan(pool, tables, contexts, queries, kv_heads * group, query_dtype=query,
                         shared_blocks=shared)
    want = attend(plan, 0, q)
    again = q.clone()
    assert attend(plan, 0, again, out=again) is again
    assert torch.equal(again.nan_to_num(7.0), want.nan_to_num(7.0))
    at = 0
    for n, m in zip(contexts, queries):
        assert torch.isfinite(again[at:at + m - 1]).all()
        at += m


def test_outputs_over_part_of_the_queries_are_refused(gpu):
    from iekv.engine.attention import AttentionPlan, attend

    pool, k, v = make_pool(12, 16, 2, 64, BF16, 96)
    plan = AttentionPlan(pool, make_tables([70, 30], 16, 12, 97), [70, 30], [2, 1], 8)
    q = queries_of(3, 8, 64, BF16, 98)
    want = attend(plan, 0, q)
    size = q.numel()
    flat = torch.zeros(8 * size, dtype=BF16, device="cuda")
    for first, to in ((0, 64), (64, 0), (0, size - 8), (2 * size, 2 * size + 512)):
        flat[first:first + size].copy_(q.flatten())
        with pytest.raises(RuntimeError, match="overlap"):
            attend(plan, 0, flat[first:first + size].view(q.shape),
                   out=flat[to:to + size].view(q.shape))
    # Heads in another order of memory over the same bytes.
    turned = flat[:size].view(8, 3, 64).permute(1, 0, 2)
    with pytest.raises(RuntimeError, match="overlap"):
        attend(plan, 0, turned, out=flat[:size].view(q.shape))
    # Beside it, and in the gap between rows that lie far apart.
    flat[:size].copy_(q.flatten())
    out = flat[size:2 * size].view(q.shape)
    assert torch.equal(attend(plan, 0, flat[:size].view(q.shape), out=out), want)
    rows = flat.view(8, size)[:6:2].narrow(1, 0, 512).view(3, 8, 64)
    rows.copy_(q)
    gap = flat[512:512 + size].view(q.shape)
    assert gap.data_ptr() + 2 * size <= rows[1].data_ptr()
    assert torch.equal(attend(plan, 0, rows, out=gap), want)
