"""Prefixes that are worth sharing, in steps of every make-up (GPU).

Tolerances as in test_gpu_attention.py. That a step shares its prefix shows in its workspace:
parts of rows that a plan without shared blocks writes whole, or more of them.
"""
from __future__ import annotations

import pytest
import torch

from test_gpu_attention import BF16, F16, F32, FP8, check, make_pool, make_tables, queries_of

pytestmark = pytest.mark.gpu

TYPES = [(BF16, BF16, 64), (BF16, FP8, 128), (F16, FP8, 64), (F16, F16, 80), (F32, F32, 32),
         (F32, F16, 64)]


def step(kv_heads, group, dim, query, cache, shared, own, queries, seed, layers=1, bs=16):
    contexts = [shared * bs + c for c in own]
    blocks = shared + sum(-(-c // bs) for c in contexts) + 2
    pool, k, v = make_pool(blocks, bs, kv_heads, dim, cache, seed, layers=layers)
    tables = make_tables(contexts, bs, blocks, seed + 1, shared)
    q = queries_of(sum(queries), kv_heads * group, dim, query, seed + 2)
    return pool, k, v, tables, contexts, q


def shares(plan, pool, tables, contexts, queries, heads, **options):
    from iekv.engine.attention import AttentionPlan

    alone = AttentionPlan(pool, tables, contexts, queries, heads, query_dtype=plan.query_dtype,
                          **options)
    return plan._workspace_bytes != alone._workspace_bytes


@pytest.mark.parametrize("query, cache, dim", TYPES)
@pytest.mark.parametrize("own, queries", [
    ([40, 300, 7, 1, 200, 90, 3, 5, 60], [1, 300, 7, 1, 150, 2, 3, 0, 1]),   # prompts among tokens
    ([5] * 40, [1] * 40),
    ([0] * 20 + [700] * 4, [1] * 24),                     # some have nothing of their own
    ([1100 + 31 * i for i in range(12)], [1] * 12),
])
def test_steps_behind_a_long_prefix(gpu, query, cache, dim, own, queries):
    kv_heads, group, shared = 8, 2, 260
    pool, k, v, tables, contexts, q = step(kv_heads, group, dim, query, cache, shared, own,
                                           queries, 100)
    _, plan = check(q, k[0], v[0], pool, tables, contexts, queries, shared_blocks=shared)
    assert shares(plan, pool, tables, contexts, queries, kv_heads * group)
    # A window that ends inside the prefix, whose first keys are sinks.
    check(q, k[0], v[0], pool, tables, contexts, queries, shared_blocks=shared, window=3001,
          sinks=17)
    check(q, k[0], v[0], pool, tables, contexts, queries, shared_blocks=shared, window=50, sinks=5)


def test_streams_and_graphs_of_shared_steps(gpu):
    """Other streams and replays give the bits of the first call, layer by layer."""
    from iekv.engine.attention import AttentionPlan, attend

    own, queries, shared = [40, 1, 7, 300, 90, 3], [1, 1, 5, 60, 1, 2], 300
    pool, k, v, tables, contexts, q = step(8, 4, 128, BF16, BF16, shared, own, queries, 110,
                                           layers=2)
    want = [check(q, k[l], v[l], pool, tables, contexts, queries, layer=l, shared_blocks=shared)[0]
            for l in range(2)]
    plan = AttentionPlan(pool, tables, contexts, queries, 32, shared_blocks=shared)
    assert shares(plan, pool, tables, contexts, queries, 32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [attend(plan, l, q) for l in range(2)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    graph, static = torch.cuda.CUDAGraph(), q.clone()
    with torch.cuda.graph(graph):
        got = [attend(plan, l, static) for l in range(2)]
    for turn in range(3):
        fresh = queries_of(q.shape[0], 32, 128, BF16, 120 + turn)
        static.copy_(fresh)
        graph.replay()
        eager = [attend(plan, l, fresh) for l in range(2)]
        torch.cuda.synchronize()
        assert all(torch.equal(g, e) for g, e in zip(got, eager))
