"""The variants that attention takes by the size of a step, against the definition in 64 bits
(GPU): workgroups of several KV heads, wide and narrow items in one launch or two, joins of
few and of many rows, caches at any address. Tolerances as in test_gpu_attention.py.
"""
from __future__ import annotations

import pytest
import torch

from test_gpu_attention import (BF16, F16, F32, FP8, check, make_pool, make_tables, queries_of,
                                reference)

pytestmark = pytest.mark.gpu


def sizes(context, n):
    return [max(1, round(context * (0.3 + 1.4 * (k + 0.5) / n))) for k in range(n)]


# 40 sequences of 4,000 tokens: a million keys of eight heads, enough for a wave to keep a
# head of its own.
@pytest.mark.parametrize("kv_heads, group, dim, bs, query, cache", [
    (8, 4, 128, 16, BF16, BF16), (8, 2, 64, 64, F16, FP8), (8, 8, 128, 16, BF16, FP8),
    (8, 1, 80, 24, F16, F16), (12, 3, 32, 16, F32, F32), (14, 2, 40, 16, F32, FP8),
    (9, 5, 16, 8, BF16, BF16), (8, 17, 24, 16, F32, BF16),
])
def test_long_streams(gpu, kv_heads, group, dim, bs, query, cache):
    contexts = sizes(4000, 40)
    blocks = sum(-(-c // bs) for c in contexts) + 2
    pool, k, v = make_pool(blocks, bs, kv_heads, dim, cache, 50)
    tables = make_tables(contexts, bs, blocks, 51)
    q = queries_of(40, kv_heads * group, dim, query, 52)
    check(q, k[0], v[0], pool, tables, contexts, [1] * 40)
    check(q, k[0], v[0], pool, tables, contexts, [1] * 40, window=3901, sinks=5)


@pytest.mark.parametrize("query, cache, dim", [(BF16, BF16, 64), (F16, FP8, 128), (F32, F32, 64)])
def test_two_tokens_of_long_streams(gpu, query, cache, dim):
    """Two query tokens a sequence, the last of which alone sees a V that is no number."""
    contexts = sizes(4000, 40)
    bs, kv_heads, group = 16, 8, 2
    blocks = sum(-(-c // bs) for c in contexts) + 2
    pool, k, v = make_pool(blocks, bs, kv_heads, dim, cache, 53)
    tables = make_tables(contexts, bs, blocks, 54)
    q = queries_of(80, kv_heads * group, dim, query, 55)
    want, plan = check(q, k[0], v[0], pool, tables, contexts, [2] * 40)
    for i in range(0, 40, 3):
        p = contexts[i] - 1
        rows = v[0].float()
        rows[tables[i][p // bs] * bs + p % bs, 1] = float("nan")
        v[0].copy_(rows.to(cache))
    from iekv.engine.attention import attend

    got = attend(plan, 0, q)
    bad = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
    for i in range(0, 40, 3):
        bad[2 * i + 1, group:2 * group] = True            # the heads of KV head 1
    assert torch.equal(torch.isnan(got), bad)
    exact, tol = reference(q, k[0], torch.nan_to_num(v[0].float()).to(cache), bs, tables, contexts,
                           [2] * 40)
    assert ((got.double() - exact).abs() <= tol)[~bad].all()


# Requests behind a prefix: a few (one launch), and as many as fill the card (two launches).
@pytest.mark.parametrize("requests, own", [(3, 5), (24, 150), (70, 300), (200, 700)])
@pytest.mark.parametrize("query, cache, dim", [(BF16, BF16, 128), (F16, FP8, 64)])
def test_streams_behind_a_prefix(gpu, requests, own, query, cache, dim):
    bs, shared, kv_heads, group = 16, 33, 8, 4
    contexts = [shared * bs + c for c in sizes(own, requests)]
    blocks = shared + sum(-(-c // bs) for c in contexts) + 2
    pool, k, v = make_pool(blocks, bs, kv_heads, dim, cache, 56)
    tables = make_tables(contexts, bs, blocks, 57, shared)
    q = queries_of(requests, kv_heads * group, dim, query, 58)
    check(q, k[0], v[0], pool, tables, contexts, [1] * requests, shared_blocks=shared)


def test_prompts_and_tokens_behind_a_prefix(gpu):
    """Sequences whose rows fill a tile read the shared keys themselves, the others together,
    whatever their order."""
    bs, shared = 16, 20
    own, queries = [40, 300, 7, 1, 200, 90, 3], [1, 300, 7, 1, 150, 2, 3]
    contexts = [shared * bs + c for c in own]
    blocks = shared + sum(-(-c // bs) for c in contexts) + 2
    for query, cache in ((BF16, BF16), (F16, FP8), (F32, F16)):
        pool, k, v = make_pool(blocks, bs, 2, 64, cache, 59)
        tables = make_tables(contexts, bs, blocks, 60, shared)
        q = queries_of(sum(queries), 8, 64, query, 61)
        check(q, k[0], v[0], pool, tables, contexts, queries, shared_blocks=shared)
        check(q, k[0], v[0], pool, tables, contexts, queries, shared_blocks=shared, window=250,
              sinks=17)


@pytest.mark.parametrize("dim", [8, 24, 32, 48, 64, 72, 96, 104, 128])
@pytest.mark.parametrize("query, cache", [(BF16, BF16), (F16, F16), (BF16, FP8)])
def test_prompts_of_caches_at_any_address(gpu, query, cache, dim):
    """A prompt's tiles come straight into LDS from aligned caches, and through registers from
    others: the same bits."""
    from iekv.engine.attention import AttentionPlan, attend
    from iekv.engine.pools import KVPool

    contexts, queries = [333, 200], [333, 70]
    pool, k, v = make_pool(36, 16, 3, dim, cache, 62)
    tables = make_tables(contexts, 16, 36, 63)
    q = queries_of(403, 9, dim, query, 64)
    want, _ = check(q, k[0], v[0], pool, tables, contexts, queries)
    odd = []
    for t in (k[0], v[0]):
        o = torch.zeros(t.numel() + 1, dtype=torch.float32, device="cuda").to(cache)[1:].view(t.shape)
        o.view(torch.uint8).copy_(t.view(torch.uint8))
        odd.append(o)
    plan = AttentionPlan(KVPool([odd[0]], [odd[1]], 16), tables, contexts, queries, 9,
                         query_dtype=query)
    assert torch.equal(attend(plan, 0, q), want)


@pytest.mark.parametrize("query, cache", [(BF16, BF16), (BF16, FP8), (F16, F16)])
def test_rows_whose_scores_rise_all_the_way(gpu, query, cache):
    """Keys whose scores grow from first to last, by less and by more than a factor of 2^8 of
    their weights a tile, and fall again: what the running maxima follow and what they do not."""
    from iekv.engine.pools import KVPool

    n, bs, dim = 900, 16, 64
    table = make_tables([n], bs, 60, 65)
    slots = (torch.tensor(table[0])[:, None] * bs + torch.arange(bs)).reshape(-1)[:n].cuda()
    for steps in (0.02, 0.2, -0.2):
        k = torch.zeros((60 * bs, 1, dim), device="cuda")
        k[slots, 0, 0] = torch.arange(n, device="cuda") * steps
        v = torch.randn((60 * bs, 1, dim), device="cuda").to(cache)
        k = k.to(cache)
        q = torch.zeros((n, 2, dim), device="cuda")
        q[:, :, 0] = 8.0
        q = q.to(query)
        check(q, k, v, KVPool([k], [v], bs), table, [n], [n])
        check(q[-1:].contiguous(), k, v, KVPool([k], [v], bs), table, [n], [1])


@pytest.mark.parametrize("query, cache", [(BF16, BF16), (F32, F32), (F16, FP8)])
def test_a_scale_of_zero_weighs_all_keys_alike(gpu, query, cache):
    contexts, queries = [140, 77], [140, 1]
    pool, k, v = make_pool(20, 16, 2, 64, cache, 66)
    tables = make_tables(contexts, 16, 20, 67)
    q = queries_of(141, 8, 64, query, 68)
    check(q, k[0], v[0], pool, tables, contexts, queries, scale=0.0)
    check(q, k[0], v[0], pool, tables, contexts, queries, scale=-0.0, window=30, sinks=2)


def test_prompts_and_tokens_behind_a_long_prefix(gpu):
    """As above behind a prefix that is worth sharing."""
    bs, shared = 16, 90
    own, queries = [40, 300, 7, 1, 200, 90, 3], [1, 300, 7, 1, 150, 2, 3]
    contexts = [shared * bs + c for c in own]
    blocks = shared + sum(-(-c // bs) for c in contexts) + 2
    for query, cache in ((BF16, BF16), (F16, FP8), (F32, F16)):
        pool, k, v = make_pool(blocks, bs, 2, 64, cache, 69)
        tables = make_tables(contexts, bs, blocks, 70, shared)
        q = queries_of(sum(queries), 8, 64, query, 71)
        check(q, k[0], v[0], pool, tables, contexts, queries, shared_blocks=shared)
        check(q, k[0], v[0], pool, tables, contexts, queries, shared_blocks=shared, window=1250,
              sinks=17)


@pytest.mark.parametrize("context", [255, 256, 257, 511, 513, 767, 769, 1023, 1025, 1300])
@pytest.mark.parametrize("query, cache, dim", [(BF16, BF16, 128), (BF16, FP8, 128), (F32, F32, 32)])
def test_contexts_around_what_one_workgroup_takes(gpu, context, query, cache, dim):
    contexts = [context, 3, context // 2]
    blocks = sum(-(-c // 16) for c in contexts) + 2
    pool, k, v = make_pool(blocks, 16, 2, dim, cache, 72)
    tables = make_tables(contexts, 16, blocks, 73)
    q = queries_of(3, 8, dim, query, 74)
    check(q, k[0], v[0], pool, tables, contexts, [1, 1, 1])
