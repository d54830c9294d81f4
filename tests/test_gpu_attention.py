"""Attention over the paged cache against the definition in 64 bits (GPU).

The tolerance of an output element is derived, not tuned. With u the largest relative error of
a rounding to the queries' type (eps / 2), A = sum_j p_j |v_j| of its row and dimension:
  - the weights may be rounded to the queries' type before the product with V: u A;
  - the output is rounded once: u |o|;
  - scores in 32 bits: a dot product of D terms is off by at most (D + 2) 2^-24 times the sum
    of its absolute products, and so the exponent's argument; a weight and the sum it is
    divided by are off by that, relative to themselves: 2 ds A;
  - the power and the sums of n terms in 32 bits: (n + 16) 2^-24 A.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16, FP8 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn


def make_pool(blocks, bs, kv_heads, dim, dtype, seed, layers=1, scale=1.0):
    from iekv.engine.pools import KVPool

    gen = torch.Generator(device="cuda").manual_seed(seed)
    k, v = ([(torch.randn((blocks * bs, kv_heads, dim), generator=gen, device="cuda") * scale)
             .to(dtype) for _ in range(layers)] for _ in range(2))
    return KVPool(k, v, bs), k, v


def make_tables(contexts, bs, blocks, seed, shared=0):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.randperm(blocks, generator=gen).tolist()
    tables, at = [], shared
    for c in contexts:
        n = max(0, -(-c // bs) - shared)
        tables.append(ids[:shared] + ids[at:at + n])
        at += n
    assert at <= blocks
    return tables


def reference(q, k, v, bs, tables, contexts, queries, window=None, sinks=0, scale=None):
    """The definition in 64 bits, and each element's tolerance."""
    d, kv_heads = q.shape[2], k.shape[1]
    group = q.shape[1] // kv_heads
    scale = 1 / math.sqrt(d) if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    outs, tols, at = [], [], 0
    for table, context, n in zip(tables, contexts, queries):
        if not n:
            continue
        slots = (torch.tensor(table, dtype=torch.long)[:, None] * bs + torch.arange(bs))
        slots = slots.reshape(-1)[:context].cuda()
        ks = k[slots].double().repeat_interleave(group, 1).permute(1, 0, 2)
        vs = v[slots].double().repeat_interleave(group, 1).permute(1, 0, 2)
        qs = q[at:at + n].double().permute(1, 0, 2)
        p = torch.arange(context - n, context, device="cuda")[:, None]
        j = torch.arange(context, device="cuda")
        seen = (j <= p) & ((j > p - (window or context + 1)) | (j < sinks))
        for lo in range(0, n, 256):
            part = slice(lo, min(n, lo + 256))
            see = seen[part]
            any_sees = see.any(0)
            kp, vp, see = ks[:, any_sees], vs[:, any_sees], see[:, any_sees]
            s = torch.matmul(qs[:, part].contiguous(), kp.transpose(1, 2).contiguous()) * scale
            size = torch.matmul(qs[:, part].abs().contiguous(),
                                kp.abs().transpose(1, 2).contiguous()) * abs(scale)
            w = torch.softmax(s.masked_fill(~see, float("-inf")), -1)
            # Masked keys take no part whatever they hold.
            vz = torch.where(torch.isfinite(vp), vp, 0.0)
            o, a = torch.matmul(w, vz), torch.matmul(w, vz.abs())
            ds = torch.where(see, size, 0.0).amax(-1, keepdim=True) * (d + 2) * 2.0 ** -24
            tol = u * a + u * o.abs() + 2 * ds * a + (see.shape[-1] + 16) * 2.0 ** -24 * a
            if q.dtype == F16:
                tol += 2.0 ** -24                       # halves a step of its subnormals
            for t, keep in ((o, outs), (tol, tols)):
                keep.append(t.permute(1, 0, 2))
        at += n
    return torch.cat(outs), torch.cat(tols)


def check(q, k, v, pool, tables, contexts, queries, layer=0, **options):
    from iekv.engine.attention import AttentionPlan, attend

    shared = options.pop("shared_blocks", 0)
    scale = options.pop("scale", None)
    plan = AttentionPlan(pool, tables, contexts, queries, q.shape[1], query_dtype=q.dtype,
                         shared_blocks=shared, **options)
    got = attend(plan, layer, q, scale=scale)
    want, tol = reference(q, k, v, pool.block_size, tables, contexts, queries, scale=scale,
                          **options)
    off = (got.double() - want).abs()
    assert got.shape == q.shape and got.dtype == q.dtype
    assert not torch.isnan(off).any()
    worst = (off / tol.clamp_min(1e-300)).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{worst} times the tolerance"
    return got, plan


def queries_of(tokens, heads, dim, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((tokens, heads, dim), generator=gen, device="cuda") * scale).to(dtype)


TYPES = [(BF16, BF16), (F16, F16), (F32, F32), (BF16, FP8), (F16, FP8), (F32, FP8), (F32, BF16),
         (F32, F16)]
# contexts, queries of a step: single tokens, prompts, chunks, odd lengths, nothing to do
STEPS = {
    "token": ([37], [1]),
    "one": ([1], [1]),
    "tokens": ([1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 700], [1] * 14),
    "prompt": ([129], [129]),
    "mixed": ([5, 0, 300, 200, 77, 64], [5, 0, 1, 131, 0, 3]),
    "long": ([5001], [1]),
}


@pytest.mark.parametrize("step", list(STEPS))
@pytest.mark.parametrize("query, cache", TYPES)
def test_types_and_lengths(gpu, query, cache, step):
    contexts, queries = STEPS[step]
    bs, kv_heads, group, dim = 16, 2, 4, 128
    blocks = sum(-(-c // bs) for c in contexts) + 3
    pool, k, v = make_pool(blocks, bs, kv_heads, dim, cache, 1)
    tables = make_tables(contexts, bs, blocks, 2)
    q = queries_of(sum(queries), kv_heads * group, dim, query, 3)
    check(q, k[0], v[0], pool, tables, contexts, queries)
    check(q, k[0], v[0], pool, tables, contexts, queries, window=48, sinks=5)


@pytest.mark.parametrize("dim", [8, 16, 24, 32, 40, 64, 72, 80, 96, 104, 120, 128])
@pytest.mark.parametrize("query, cache", [(BF16, BF16), (F16, FP8), (F32, F32)])
def test_head_sizes(gpu, query, cache, dim):
    contexts, queries = [200, 90, 33], [1, 70, 33]
    bs, kv_heads, group = 16, 3, 2
    pool, k, v = make_pool(30, bs, kv_heads, dim, cache, 4)
    tables = make_tables(contexts, bs, 30, 5)
    q = queries_of(sum(queries), kv_heads * group, dim, query, 6)
    check(q, k[0], v[0], pool, tables, contexts, queries, window=50, sinks=3)


@pytest.mark.parametrize("kv_heads, group", [(1, 1), (1, 7), (5, 3), (2, 16), (1, 17), (1, 71),
                                             (1, 128), (8, 8), (13, 1)])
def test_head_layouts(gpu, kv_heads, group):
    contexts, queries = [150, 41], [2, 41]
    for dim, query, cache in ((64, BF16, BF16), (80, F32, F16)):
        pool, k, v = make_pool(16, 16, kv_heads, dim, cache, 7)
        tables = make_tables(contexts, 16, 16, 8)
        q = queries_of(sum(queries), kv_heads * group, dim, query, 9)
        check(q, k[0], v[0], pool, tables, contexts, queries)


@pytest.mark.parametrize("bs", [1, 3, 5, 8, 16, 24, 48, 64, 100, 256])
def test_block_sizes(gpu, bs):
    contexts, queries = [190, 1, 300], [1, 1, 170]
    blocks = sum(-(-c // bs) for c in contexts) + 2
    pool, k, v = make_pool(blocks, bs, 2, 64, F16, 10)
    tables = make_tables(contexts, bs, blocks, 11)
    q = queries_of(sum(queries), 8, 64, F16, 12)
    check(q, k[0], v[0], pool, tables, contexts, queries)
    check(q, k[0], v[0], pool, tables, contexts, queries, window=70, sinks=9)


@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (2, 64), (7, 0), (64, 4), (100, 100),
                                           (299, 1), (300, 0), (1000, 4), (40, 1000), (None, 7),
                                           (1 << 50, 1 << 50)])
@pytest.mark.parametrize("query", [BF16, F32])
def test_windows_and_sinks(gpu, window, sinks, query):
    contexts, queries = [300, 299, 64, 10], [300, 1, 5, 10]
    pool, k, v = make_pool(60, 16, 2, 64, query, 13)
    tables = make_tables(contexts, 16, 60, 14)
    q = queries_of(sum(queries), 6, 64, query, 15)
    options = dict(window=window, sinks=sinks)
    check(q, k[0], v[0], pool, tables, contexts, queries, **options)


@pytest.mark.parametrize("shared, contexts, queries", [
    (4, [65, 100, 64, 300], [1, 36, 0, 1]),
    (4, [64, 64, 64], [1, 1, 1]),                    # nothing of their own
    (4, [70, 64, 90], [40, 64, 26]),                 # queries inside the prefix
    (1, [17] * 40, [1] * 40),
    (128, [2049 + 31 * i for i in range(20)], [1] * 20),
    (100, [1700, 1601, 1650], [100, 1, 50]),
    (3, [100], [1]),
])
@pytest.mark.parametrize("query, cache", [(BF16, BF16), (F16, FP8), (F32, F32)])
def test_shared_prefixes(gpu, query, cache, shared, contexts, queries):
    bs = 16
    blocks = shared + sum(-(-c // bs) for c in contexts) + 3
    pool, k, v = make_pool(blocks, bs, 2, 64, cache, 16)
    tables = make_tables(contexts, bs, blocks, 17, shared)
    q = queries_of(sum(queries), 8, 64, query, 18)
    check(q, k[0], v[0], pool, tables, contexts, queries, shared_blocks=shared)
    check(q, k[0], v[0], pool, tables, contexts, queries, shared_blocks=shared, window=40, sinks=5)


@pytest.mark.parametrize("query, cache", [(BF16, BF16), (F32, F32), (BF16, FP8)])
def test_what_masked_places_hold_stays_out(gpu, query, cache):
    """Cache rows that no query may see (before the window, behind the context, in blocks of
    nobody) and rows that only other queries see hold NaN and infinities."""
    from iekv.engine.attention import AttentionPlan, attend

    bs, window, sinks = 16, 40, 3
    contexts, queries = [200, 90], [1, 1]
    pool, k, v = make_pool(24, bs, 2, 64, cache, 19)
    tables = make_tables(contexts, bs, 24, 20)
    bad = torch.ones(24 * bs, dtype=torch.bool, device="cuda")
    for table, context in zip(tables, contexts):
        for j in list(range(sinks)) + list(range(context - window, context)):
            bad[table[j // bs] * bs + j % bs] = False
    worst = float("nan") if cache == FP8 else float("inf")
    for t in (k[0], v[0]):
        rows = t.float()
        rows[bad] = float("nan")
        rows[bad.nonzero()[::2, 0]] = worst
        t.copy_(rows.to(cache))
    q = queries_of(2, 8, 64, query, 21)
    got, _ = check(q, k[0], v[0], pool, tables, contexts, queries, window=window, sinks=sinks)
    assert torch.isfinite(got).all()

    # A prompt: the last token's V is not a number. Only its own row may show it; and K's
    # likewise.
    for which in (k, v):
        pool, k, v = make_pool(24, bs, 2, 64, cache, 22)
        n = 150
        table = make_tables([n], bs, 24, 23)
        slot = table[0][(n - 1) // bs] * bs + (n - 1) % bs
        q = queries_of(n, 8, 64, query, 24)
        plan = AttentionPlan(pool, table, [n], [n], 8, query_dtype=query)
        before = attend(plan, 0, q)
        target = (k if which is not v else v)[0]
        rows = target.float()
        rows[slot] = float("nan")
        target.copy_(rows.to(cache))
        got = attend(plan, 0, q)
        want, tol = reference(q[:-1], k[0], v[0], bs, table, [n - 1], [n - 1])
        assert ((got[:-1].double() - want).abs() <= tol).all()
        assert torch.isnan(got[-1]).any()
        assert torch.isfinite(before).all()


def test_large_scores(gpu):
    """Scores far apart: one key takes all, and nothing overflows."""
    for query in (BF16, F16, F32):
        contexts, queries = [150, 90], [1, 90]
        pool, k, v = make_pool(20, 16, 2, 64, query, 25, scale=30.0)
        tables = make_tables(contexts, 16, 20, 26)
        q = queries_of(91, 8, 64, query, 27, scale=30.0)
        check(q, k[0], v[0], pool, tables, contexts, queries)
        check(q, k[0], v[0], pool, tables, contexts, queries, scale=-0.3)


def test_strides_and_addresses(gpu):
    """Queries that are slices of wider rows, at odd offsets, with heads in another order of
    memory; caches that begin at odd elements."""
    from iekv.engine.attention import AttentionPlan, attend
    from iekv.engine.pools import KVPool

    contexts, queries = [70, 200], [5, 1]
    for query in (BF16, F32):
        pool, k, v = make_pool(20, 16, 2, 64, query, 28)
        tables = make_tables(contexts, 16, 20, 29)
        q = queries_of(6, 8, 64, query, 30)
        want, plan = check(q, k[0], v[0], pool, tables, contexts, queries)
        fused = torch.zeros((6, 8 * 64 + 2 * 2 * 64 + 1), dtype=query, device="cuda")
        fused[:, 1:513] = q.view(6, 512)
        assert torch.equal(attend(plan, 0, fused[:, 1:513].view(6, 8, 64)), want)
        assert torch.equal(attend(plan, 0, q.permute(1, 0, 2).contiguous().permute(1, 0, 2)), want)
        assert torch.equal(attend(plan, 0, q.permute(0, 2, 1).contiguous().permute(0, 2, 1)), want)
        flat = torch.zeros(k[0].numel() + 1, dtype=query, device="cuda")
        odd = []
        for t in (k[0], v[0]):
            o = flat.clone()[1:].view(t.shape)
            o.copy_(t)
            odd.append(o)
        other = AttentionPlan(KVPool([odd[0]], [odd[1]], 16), tables, contexts, queries, 8)
        assert torch.equal(attend(other, 0, q), want)
        out = torch.empty_like(q)
        assert attend(plan, 0, q, out=out) is out and torch.equal(out, want)
        # Overwritten queries with the same result in place.
        again = q.clone()
        assert torch.equal(attend(plan, 0, again, out=torch.empty_like(q)), want)


def test_offsets_past_32_bits(gpu):
    """A cache of more than 2^31 elements and 2^32 bytes: blocks at its end."""
    from iekv.engine.pools import KVPool

    bs, kv_heads, dim = 16, 8, 128
    blocks = (1 << 31) // (bs * kv_heads * dim) + 64
    shape = (blocks * bs, kv_heads, dim)
    k, v = (torch.zeros(shape, dtype=BF16, device="cuda") for _ in range(2))
    contexts, queries = [500, 100], [1, 100]
    tables = [[blocks - 1 - 2 * i for i in range(32)], [blocks - 2 - 2 * i for i in range(7)]]
    for t in (k, v):
        t[-80 * bs:].normal_()
    pool = KVPool([k], [v], bs)
    q = queries_of(101, 32, dim, BF16, 31)
    check(q, k, v, pool, tables, contexts, queries)


def test_layers_streams_graphs_and_repeats(gpu):
    from iekv.engine.attention import AttentionPlan, attend

    contexts, queries = [1500, 1200, 1100], [1, 1, 40]
    bs = 16
    blocks = sum(-(-c // bs) for c in contexts) + 64
    pool, k, v = make_pool(blocks, bs, 2, 128, BF16, 32, layers=3)
    tables = make_tables(contexts, bs, blocks, 33, shared=60)
    q = queries_of(42, 8, 128, BF16, 34)
    for options in (dict(), dict(shared_blocks=60), dict(window=600, sinks=4)):
        want = [check(q, k[l], v[l], pool, tables, contexts, queries, layer=l, **options)[0]
                for l in range(3)]
        plan = AttentionPlan(pool, tables, contexts, queries, 8, **options)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [attend(plan, l, q) for l in range(3)]
        torch.cuda.current_stream().wait_stream(side)
        for g, w in zip(got, want):
            assert torch.equal(g, w)            # the same bits, whatever the stream
        graph = torch.cuda.CUDAGraph()
        static = q.clone()
        with torch.cuda.graph(graph):
            got = [attend(plan, l, static) for l in range(3)]
        for turn in range(3):
            fresh = queries_of(42, 8, 128, BF16, 35 + turn)
            static.copy_(fresh)
            graph.replay()
            eager = [attend(plan, l, fresh) for l in range(3)]
            torch.cuda.synchronize()
            for g, w in zip(got, eager):
                assert torch.equal(g, w)


def test_refusals(gpu):
    from iekv.engine.attention import AttentionPlan, attend
    from iekv.engine.pools import KVPool

    pool, k, v = make_pool(8, 16, 2, 64, BF16, 40, layers=2)
    args = ([[1, 2], [3]], [20, 5], [1, 5], 8)
    plan = AttentionPlan(pool, *args)
    q = queries_of(6, 8, 64, BF16, 41)
    attend(plan, 1, q)
    with pytest.raises(IndexError, match="out of range"):
        AttentionPlan(pool, [[1, 8], [3]], *args[1:])
    with pytest.raises(IndexError, match="out of range"):
        AttentionPlan(pool, [[1, 1 << 40], [3]], *args[1:])
    with pytest.raises(IndexError, match="needs 2 blocks"):
        AttentionPlan(pool, [[1], [3]], *args[1:])
    with pytest.raises(TypeError):
        AttentionPlan(pool, [[1, 2.5], [3]], *args[1:])
    with pytest.raises(TypeError):
        AttentionPlan(pool, [torch.tensor([1, 2]).cuda(), [3]], *args[1:])
    with pytest.raises(ValueError, match="3 block tables"):
        AttentionPlan(pool, [[1, 2], [3], [4]], *args[1:])
    with pytest.raises(ValueError, match="window"):
        AttentionPlan(pool, *args, window=0)
    with pytest.raises(ValueError, match="begin with"):
        AttentionPlan(pool, [[1, 2], [3]], [20, 16], [1, 5], 8, shared_blocks=1)
    with pytest.raises(ValueError, match="does not fill"):
        AttentionPlan(pool, [[1, 2], [1]], [20, 5], [1, 5], 8, shared_blocks=1)
    with pytest.raises(RuntimeError, match="7 query heads"):
        AttentionPlan(pool, *args[:3], 7)
    with pytest.raises(RuntimeError, match="queries in a context"):
        AttentionPlan(pool, [[1, 2], [3]], [20, 5], [1, 6], 8)
    with pytest.raises(RuntimeError, match="type"):
        AttentionPlan(pool, *args, query_dtype=F16)
    with pytest.raises(ValueError, match="float64"):
        AttentionPlan(pool, *args, query_dtype=torch.float64)
    with pytest.raises(ValueError, match="queries of"):
        attend(plan, 0, q.float())
    with pytest.raises(ValueError, match="queries of"):
        attend(plan, 0, q.cpu())
    with pytest.raises(ValueError, match="shape"):
        attend(plan, 0, q[:5])
    with pytest.raises(IndexError):
        attend(plan, 2, q)
    with pytest.raises(RuntimeError, match="backward"):
        attend(plan, 0, q.clone().requires_grad_())
    with pytest.raises(ValueError, match="out"):
        attend(plan, 0, q, out=torch.empty_like(q).float())
    with pytest.raises(RuntimeError, match="scale"):
        attend(plan, 0, q, scale=float("inf"))
    odd = torch.zeros((16, 2, 12), dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError, match="head_dim 12"):
        AttentionPlan(KVPool([odd], [odd.clone()], 16), [[0]], [1], [1], 2)
    flat = torch.zeros((16, 64), dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="caches of"):
        AttentionPlan(KVPool([flat], [flat.clone()], 16), [[0]], [1], [1], 2)
    # An empty step is a step.
    empty = AttentionPlan(pool, [], [], [], 8)
    assert attend(empty, 0, q[:0]).shape == (0, 8, 64)
    nothing = AttentionPlan(pool, [[1], []], [5, 0], [0, 0], 8)
    assert attend(nothing, 0, q[:0]).shape == (0, 8, 64)
    # NumPy tables and padded ones are as good as lists.
    import numpy as np

    same = AttentionPlan(pool, np.array([[1, 2, -1], [3, -1, -1]]), np.array([20, 5]),
                         np.array([1, 5]), 8)
    assert torch.equal(attend(same, 0, q), attend(plan, 0, q))
