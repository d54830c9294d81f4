"""What attention computes where a number format ends, against the definition in 64 bits (GPU).

Tolerances are derived as in test_gpu_attention.py. With u the largest relative error of a
rounding to the queries' type and A = sum_j p_j |v_j| of an output element: single tokens hold
their weights in two parts of the queries' type, so that a weight is off by u^2 of itself (u of
a remainder that is at most u of it), and their products are twice as many terms.
"""
from __future__ import annotations

import pytest
import torch

from test_gpu_attention import BF16, F16, FP8, F32, make_pool, make_tables, queries_of

pytestmark = pytest.mark.gpu


def attention(q, k, v, position, scale, window=None):
    """One KV head in 64 bits: q [rows, D] at ``position`` [rows], k and v [n, D]. The output,
    A and the largest |score| that a row's weights are taken of."""
    q, k, v = q.double(), k.double(), v.double()
    j = torch.arange(k.shape[0], device="cuda")
    seen = j <= position[:, None]
    if window is not None:
        seen &= j > position[:, None] - window
    s = torch.matmul(q, k.t().contiguous()) * scale
    size = torch.matmul(q.abs(), k.abs().t().contiguous()) * abs(scale)
    w = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
    return torch.matmul(w, v), torch.matmul(w, v.abs()), \
        torch.where(seen, size, 0.0).amax(-1, keepdim=True)


@pytest.mark.parametrize("query, cache", [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8)])
@pytest.mark.parametrize("contexts", [[300, 64, 1, 33], [5001]])
def test_weights_of_single_tokens_keep_their_bits(gpu, query, cache, contexts):
    """Of an output that is near zero beside its terms, rounded weights would be most of the
    error."""
    from iekv.engine.attention import AttentionPlan, attend

    bs, kv_heads, group, dim = 16, 2, 4, 64
    blocks = sum(-(-c // bs) for c in contexts) + 2
    pool, k, v = make_pool(blocks, bs, kv_heads, dim, cache, 80)
    tables = make_tables(contexts, bs, blocks, 81)
    q = queries_of(len(contexts), kv_heads * group, dim, query, 82)
    plan = AttentionPlan(pool, tables, contexts, [1] * len(contexts), kv_heads * group,
                         query_dtype=query)
    got = attend(plan, 0, q).double()
    u = torch.finfo(query).eps / 2
    for i, (table, n) in enumerate(zip(tables, contexts)):
        slots = (torch.tensor(table)[:, None] * bs + torch.arange(bs)).reshape(-1)[:n].cuda()
        for h in range(kv_heads):
            rows = slice(h * group, (h + 1) * group)
            o, a, size = attention(q[i, rows], k[0][slots, h], v[0][slots, h],
                                   torch.full((group,), n - 1, device="cuda"), dim ** -0.5)
            ds = size * (dim + 2) * 2.0 ** -24
            tol = u * o.abs() + (u * u + 2 * ds + (2 * n + 16) * 2.0 ** -24) * a
            if query == F16:
                tol += 2.0 ** -24
            assert ((got[i, rows] - o).abs() <= tol).all()


def tail(v, hot_v, counts, score):
    """Output and A of a key of weight one and ``counts`` keys of e^-score beside it, whose
    values' sums (and sums of absolute values) are ``v``."""
    import math

    w = math.exp(-score)
    total = 1.0 + counts.double() * w
    return tuple((h + w * s) / total for h, s in zip((hot_v, hot_v.abs()), v))


# A key 17 nats above 60,000 others, whose weights are below half of float16's smallest number.
TAIL, SCORE = 60000, 17.375


@pytest.mark.parametrize("hot", [0.0, 0.25])
@pytest.mark.parametrize("query, cache", [(F16, F16), (F16, FP8), (BF16, BF16), (F32, F32)])
def test_a_long_tail_counts_for_single_tokens(gpu, query, cache, hot):
    """800 sequences over one table: enough for a wave to take a whole context."""
    from iekv.engine.attention import AttentionPlan, attend
    from iekv.engine.pools import KVPool

    bs, kv_heads, dim, n = 16, 4, 64, TAIL + 1
    blocks = -(-n // bs)
    k = torch.zeros((blocks * bs, kv_heads, dim), device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(83)
    v = (torch.rand(k.shape, generator=gen, device="cuda") + 0.5).to(cache)
    k[5, :, 0] = SCORE * (2 if cache == FP8 else 1)      # 34.75 is no fp8 number, 36 is
    k, v[5] = k.to(cache), torch.full((kv_heads, dim), hot, device="cuda").to(cache)
    score = k[5, 0, 0].item() * (0.5 if cache == FP8 else 1)
    q = torch.zeros((800, kv_heads, dim), dtype=query, device="cuda")
    q[:, :, 0] = 1.0
    plan = AttentionPlan(KVPool([k], [v], bs), [list(range(blocks))] * 800, [n] * 800, [1] * 800,
                         kv_heads, query_dtype=query)
    got = attend(plan, 0, q, scale=0.5 if cache == FP8 else 1.0).double()
    assert torch.equal(got, got[:1].expand_as(got))
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[5] = False
    sums = v[:n][rest].double().sum(0)
    o, a = tail((sums, sums), v[5].double(), torch.tensor(TAIL, device="cuda"), score)
    u = torch.finfo(query).eps / 2
    ds = score * (dim + 2) * 2.0 ** -24
    tol = u * o + (u * u + 2 * ds + (2 * n + 16) * 2.0 ** -24) * a + (2.0 ** -24 if query == F16
                                                                      else 0.0)
    assert ((got[0] - o).abs() <= tol).all()


@pytest.mark.parametrize("hot", [0.0, 0.25])
@pytest.mark.parametrize("query, cache", [(F16, F16), (F16, FP8), (BF16, BF16)])
def test_a_long_tail_counts_for_prompts(gpu, query, cache, hot):
    """512 queries of eight KV heads: as many workgroups as take a context in one piece.
    float16 weights are steps of 2^-24 there, 2^7 or more times the weights."""
    from iekv.engine.attention import AttentionPlan, attend
    from iekv.engine.pools import KVPool

    bs, kv_heads, group, dim, n, queries = 16, 8, 4, 64, TAIL + 1, 512
    blocks = -(-n // bs)
    k = torch.zeros((blocks * bs, kv_heads, dim), device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(84)
    v = (torch.rand(k.shape, generator=gen, device="cuda") + 0.5).to(cache)
    k[0, :, 0] = SCORE * (2 if cache == FP8 else 1)
    k, v[0] = k.to(cache), torch.full((kv_heads, dim), hot, device="cuda").to(cache)
    score = k[0, 0, 0].item() * (0.5 if cache == FP8 else 1)
    q = torch.zeros((queries, kv_heads * group, dim), dtype=query, device="cuda")
    q[:, :, 0] = 1.0
    plan = AttentionPlan(KVPool([k], [v], bs), [list(range(blocks))], [n], [queries],
                         kv_heads * group, query_dtype=query)
    got = attend(plan, 0, q, scale=0.5 if cache == FP8 else 1.0).double()
    got = got.view(queries, kv_heads, group, dim)
    sums = v[1:n].double().cumsum(0)[-queries:]
    counts = torch.arange(n - queries, n, device="cuda")[:, None, None]
    o, a = tail((sums, sums), v[0].double(), counts, score)
    u = torch.finfo(query).eps / 2
    ds = score * (dim + 2) * 2.0 ** -24
    tol = u * o + (u + 2 * ds + (n + 16) * 2.0 ** -24) * a
    if query == F16:
        tol = tol + 2.0 ** -24 + 2.0 ** -25 / 2 ** 7 * sums
    assert ((got - o[:, :, None]).abs() <= tol[:, :, None]).all()


@pytest.mark.parametrize("query, cache, size", [(F16, F16, 6e4), (BF16, BF16, 1e6),
                                                (F32, F32, 1e8), (F32, F16, 6e4)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("contexts, queries", [([150], [150]), ([5001, 40], [1, 1]),
                                               ([1500, 900], [700, 2])])
def test_scores_far_past_24_bits(gpu, query, cache, size, sign, contexts, queries):
    """Finite scores between whose neighbours in 32 bits lie many powers of e: the largest takes
    all, and its row is its V to the bit."""
    from iekv.engine.attention import AttentionPlan, attend

    bs, kv_heads, group, dim = 16, 2, 4, 64
    blocks = sum(-(-c // bs) for c in contexts) + 2
    pool, k, v = make_pool(blocks, bs, kv_heads, dim, cache, 85)
    tables = make_tables(contexts, bs, blocks, 86)
    k[0].zero_()
    gen = torch.Generator(device="cuda").manual_seed(87)
    k[0][:, :, 0] = (torch.rand(k[0].shape[:2], generator=gen, device="cuda") * -size).to(cache)
    for table in tables:
        k[0][table[0] * bs + 3, :, 0] = size
    q = torch.zeros((sum(queries), kv_heads * group, dim), dtype=query, device="cuda")
    q[:, :, 0] = size * sign
    plan = AttentionPlan(pool, tables, contexts, queries, kv_heads * group, query_dtype=query)
    got = attend(plan, 0, q, scale=sign * dim ** -0.5)
    at = 0
    for table, n, m in zip(tables, contexts, queries):
        first = max(0, 3 - (n - m))              # queries before the key do not see it
        want = v[0][table[0] * bs + 3].to(query).repeat_interleave(group, 0)
        assert torch.equal(got[at + first:at + m], want.expand(m - first, -1, -1))
        assert torch.isfinite(got[at:at + m]).all()
        at += m
