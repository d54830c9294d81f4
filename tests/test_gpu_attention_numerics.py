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
