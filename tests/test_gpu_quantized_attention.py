"""Attention over microscaled caches against the definition in 64 bits (GPU).

The keys and values are those that the records stand for, in the queries' type. From there the
tolerances are those of test_gpu_attention.py, whose derivation holds whatever the cache: the
conversion to the queries' type is exact, or rounds to what the definition is given.
"""
from __future__ import annotations

import pytest
import torch

from quantized_reference import FORMATS, decode, encode
from test_gpu_attention import BF16, F16, F32, STEPS, make_tables, queries_of, reference

pytestmark = pytest.mark.gpu

TYPES = [BF16, F16, F32]


def make_pool(blocks, bs, kv_heads, dim, format, query, seed, layers=1, scale=1.0, rows=None):
    """A pool of random rows, and K and V of each layer as the queries' type holds them."""
    from iekv.engine.quantized import QuantizedPool

    gen = torch.Generator().manual_seed(seed)
    caches, values = [], []
    for _ in range(2 * layers):
        x = torch.randn((blocks * bs, kv_heads, dim), generator=gen) * scale
        x *= torch.exp2(torch.randn((kv_heads, dim), generator=gen))
        if rows is not None:
            x = rows(x)
        record = encode(x, format)
        caches.append(record.cuda())
        values.append(decode(record, format).to(F32).to(query).cuda())
    pool = QuantizedPool(caches[:layers], caches[layers:], bs, format)
    return pool, values[:layers], values[layers:]


def check(q, k, v, pool, tables, contexts, queries, layer=0, shared_blocks=0, scale=None,
          **options):
    from iekv.engine.attention import AttentionPlan, attend

    plan = AttentionPlan(pool, tables, contexts, queries, q.shape[1], query_dtype=q.dtype,
                         shared_blocks=shared_blocks, **options)
    got = attend(plan, layer, q, scale=scale)
    want, tol = reference(q, k, v, pool.block_size, tables, contexts, queries, scale=scale,
                          **options)
    # Small weights end somewhere, which counts where the V of the large ones are zeros. The power
    # is zero below 2^-126. float16 ends at 2^-24, and rounds by 2^-25: its weights are held 2^7
    # or more above their size, so that each is off by 2^-32 of the largest at most, which is one
    # of those that the sum, at least as large, divides. Each of n keys: n times that times |v|.
    lost = 2.0 ** -32 if q.dtype == F16 else 2.0 ** -126
    tol = tol + lost * max(contexts) * v.double().abs().amax()
    off = (got.double() - want).abs()
    assert got.shape == q.shape and got.dtype == q.dtype
    assert not torch.isnan(off).any()
    worst = (off / tol.clamp_min(1e-300)).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{worst} times the tolerance"
    return got, plan


@pytest.mark.parametrize("step", list(STEPS))
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("query", TYPES, ids=str)
def test_types_and_lengths(gpu, query, format, step):
    contexts, queries = STEPS[step]
    bs, kv_heads, group, dim = 16, 2, 4, 128
    blocks = sum(-(-c // bs) for c in contexts) + 3
    pool, k, v = make_pool(blocks, bs, kv_heads, dim, format, query, 1)
    tables = make_tables(contexts, bs, blocks, 2)
    q = queries_of(sum(queries), kv_heads * group, dim, query, 3)
    check(q, k[0], v[0], pool, tables, contexts, queries)
    check(q, k[0], v[0], pool, tables, contexts, queries, window=48, sinks=5)


@pytest.mark.parametrize("dim", [8, 16, 24, 32, 40, 48, 56, 64, 72, 80, 88, 96, 104, 112, 120,
                                 128])
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("query", TYPES, ids=str)
def test_head_sizes(gpu, query, format, dim):
    """Heads that end inside a group, a load and a lane's share; records of the pool's last row
    among them, behind which nothing may be read."""
    contexts, queries = [200, 90, 33], [1, 70, 33]
    bs, kv_heads, group = 16, 3, 2
    pool, k, v = make_pool(22, bs, kv_heads, dim, format, query, 4)
    tables = make_tables(contexts, bs, 22, 5)
    assert 21 in sum(tables, [])
    q = queries_of(sum(queries), kv_heads * group, dim, query, 6)
    check(q, k[0], v[0], pool, tables, contexts, queries, window=50, sinks=3)


@pytest.mark.parametrize("kv_heads, group", [(1, 1), (1, 7), (5, 3), (2, 16), (1, 17), (1, 71),
                                             (1, 128), (8, 8), (13, 1)])
@pytest.mark.parametrize("format", FORMATS)
def test_head_layouts(gpu, kv_heads, group, format):
    contexts, queries = [150, 41], [2, 41]
    for dim, query in ((64, BF16), (80, F32)):
        pool, k, v = make_pool(16, 16, kv_heads, dim, format, query, 7)
        tables = make_tables(contexts, 16, 16, 8)
        q = queries_of(sum(queries), kv_heads * group, dim, query, 9)
        check(q, k[0], v[0], pool, tables, contexts, queries)


@pytest.mark.parametrize("bs", [1, 3, 5, 8, 24, 64, 100, 256])
@pytest.mark.parametrize("format", FORMATS)
def test_block_sizes(gpu, bs, format):
    contexts, queries = [190, 1, 300], [1, 1, 170]
    blocks = sum(-(-c // bs) for c in contexts) + 2
    pool, k, v = make_pool(blocks, bs, 2, 64, format, F16, 10)
    tables = make_tables(contexts, bs, blocks, 11)
    q = queries_of(sum(queries), 8, 64, F16, 12)
    check(q, k[0], v[0], pool, tables, contexts, queries)
    check(q, k[0], v[0], pool, tables, contexts, queries, window=70, sinks=9)


@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (2, 64), (64, 4), (299, 1), (40, 1000),
                                           (None, 7)])
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("query", [BF16, F32], ids=str)
def test_windows_and_sinks(gpu, window, sinks, query, format):
    contexts, queries = [300, 299, 64, 10], [300, 1, 5, 10]
    pool, k, v = make_pool(60, 16, 2, 64, format, query, 13)
    tables = make_tables(contexts, 16, 60, 14)
    q = queries_of(sum(queries), 6, 64, query, 15)
    check(q, k[0], v[0], pool, tables, contexts, queries, window=window, sinks=sinks)


@pytest.mark.parametrize("shared, contexts, queries", [
    (4, [65, 100, 64, 300], [1, 36, 0, 1]),
    (4, [70, 64, 90], [40, 64, 26]),
    (256, [4097 + 31 * i for i in range(24)], [1] * 24),
])
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("query", TYPES, ids=str)
def test_shared_prefixes(gpu, query, format, shared, contexts, queries):
    bs = 16
    blocks = shared + sum(-(-c // bs) - shared for c in contexts) + 3
    pool, k, v = make_pool(blocks, bs, 4, 64, format, query, 16)
    tables = make_tables(contexts, bs, blocks, 17, shared)
    q = queries_of(sum(queries), 16, 64, query, 18)
    check(q, k[0], v[0], pool, tables, contexts, queries, shared_blocks=shared)


@pytest.mark.parametrize("kv_heads, dim, query", [
    (1, 128, BF16), (2, 128, BF16), (4, 128, F16), (6, 128, BF16), (8, 128, BF16), (8, 128, F32),
    (4, 96, BF16), (12, 64, F16), (4, 32, BF16), (4, 64, F32), (8, 80, BF16), (4, 120, F16)])
@pytest.mark.parametrize("format", FORMATS)
def test_long_streams(gpu, kv_heads, dim, query, format):
    """Steps whose workgroups take several heads, whose items are cut into parts, and both;
    blocks that are in several tables and several times in one; a window that starts anywhere
    in a block."""
    contexts = [20000 // kv_heads + 131 * i for i in range(64)]
    bs, blocks = 16, 150
    assert sum(contexts) * kv_heads > 4 * 256 * 4 * 256      # long: of four heads together
    pool, k, v = make_pool(blocks, bs, kv_heads, dim, format, query, 19)
    gen = torch.Generator().manual_seed(20)
    tables = [torch.randint(blocks, (-(-c // bs),), generator=gen).tolist() for c in contexts]
    q = queries_of(64, 4 * kv_heads, dim, query, 21)
    check(q, k[0], v[0], pool, tables, contexts, [1] * 64)
    check(q[:32], k[0], v[0], pool, tables[32:], contexts[32:], [1] * 32, window=4001, sinks=5)


@pytest.mark.parametrize("query", [BF16, F32], ids=str)
@pytest.mark.parametrize("format", FORMATS)
def test_streams_of_middle_length_and_a_chunk(gpu, query, format):
    """Long enough for heads to be taken together, alone and beside a prompt's chunk."""
    contexts = [4000 + 131 * i for i in range(16)]
    assert 4 * 256 * 256 < sum(contexts) * 4 < 4 * 4 * 256 * 256
    pool, k, v = make_pool(150, 16, 4, 128, format, query, 57)
    gen = torch.Generator().manual_seed(58)
    tables = [torch.randint(150, (-(-c // 16),), generator=gen).tolist() for c in contexts]
    q = queries_of(16 + 299, 16, 128, query, 59)
    check(q[:16], k[0], v[0], pool, tables, contexts, [1] * 16)
    check(q, k[0], v[0], pool, tables, contexts, [1] * 15 + [300])


@pytest.mark.parametrize("group, queries, query, window", [
    (4, 3, BF16, None), (4, 4, BF16, 3000), (7, 2, F16, None), (1, 5, F32, 77), (20, 1, F32, None)])
@pytest.mark.parametrize("format", FORMATS)
def test_long_streams_of_several_rows(gpu, group, queries, query, window, format):
    """Rows of several tokens, whose masks end a stream differently; more heads in a group than a
    workgroup holds; a captured call that is replayed among eager ones."""
    from iekv.engine.attention import attend

    contexts = [5000 + 131 * i for i in range(64)]
    pool, k, v = make_pool(150, 16, 4, 64, format, query, 54)
    gen = torch.Generator().manual_seed(55)
    tables = [torch.randint(150, (-(-c // 16),), generator=gen).tolist() for c in contexts]
    q = queries_of(64 * queries, 4 * group, 64, query, 56)
    want, plan = check(q, k[0], v[0], pool, tables, contexts, [queries] * 64,
                       **({} if window is None else dict(window=window, sinks=3)))
    side, now, out = torch.cuda.Stream(), torch.zeros_like(q), torch.empty_like(q)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attend(plan, 0, now, out=out)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(plan, 0, now, out=out)
    for x in (q, -q, q):
        now.copy_(x)
        graph.replay()
        replayed = out.clone()
        assert torch.equal(replayed, attend(plan, 0, x))
        torch.cuda.synchronize()
    assert torch.equal(replayed, want)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("query", TYPES, ids=str)
def test_long_streams_at_any_address(gpu, query, format):
    """Caches that begin at a multiple of 16 bytes, of 4, and at an odd byte; the output in the
    queries' place."""
    from iekv.engine.attention import AttentionPlan, attend
    from iekv.engine.quantized import QuantizedPool

    contexts = [5000 + 131 * i for i in range(64)]
    pool, k, v = make_pool(150, 16, 4, 64, format, query, 51)
    gen = torch.Generator().manual_seed(52)
    tables = [torch.randint(150, (-(-c // 16),), generator=gen).tolist() for c in contexts]
    q = queries_of(64, 12, 64, query, 53)
    check(q, k[0], v[0], pool, tables, contexts, [1] * 64)
    for first, second in ((16, 16), (4, 0), (0, 4), (1, 3)):
        arrays = []
        for t, skip in zip(pool._arrays, (first, second)):
            o = torch.zeros(t.numel() + skip, dtype=torch.uint8, device="cuda")[skip:].view(t.shape)
            o.copy_(t)
            arrays.append(o)
        moved = QuantizedPool(arrays[:1], arrays[1:], 16, format)
        want, plan = check(q, k[0], v[0], moved, tables, contexts, [1] * 64)
        again = q.clone()
        assert attend(plan, 0, again, out=again) is again and torch.equal(again, want)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("query", TYPES, ids=str)
def test_what_masked_places_hold_stays_out(gpu, query, format):
    """Rows that no query may see hold groups that are no numbers; so, in a prompt, does the
    last token's V or K, which only its own row may show."""
    from iekv.engine.attention import AttentionPlan, attend

    bs, window, sinks = 16, 40, 3
    contexts, queries = [200, 90], [1, 1]
    pool, k, v = make_pool(24, bs, 2, 64, format, query, 22)
    tables = make_tables(contexts, bs, 24, 23)
    bad = torch.ones(24 * bs, dtype=torch.bool, device="cuda")
    for table, context in zip(tables, contexts):
        for j in list(range(sinks)) + list(range(context - window, context)):
            bad[table[j // bs] * bs + j % bs] = False
    for t in pool._arrays:
        t[bad, :, -4:] = 255
    q = queries_of(2, 8, 64, query, 24)
    got, _ = check(q, k[0], v[0], pool, tables, contexts, queries, window=window, sinks=sinks)
    assert torch.isfinite(got).all()
    for which in (0, 1):
        n = 150
        pool, k, v = make_pool(24, bs, 2, 64, format, query, 25)
        table = make_tables([n], bs, 24, 26)
        slot = table[0][(n - 1) // bs] * bs + (n - 1) % bs
        q = queries_of(n, 8, 64, query, 27)
        plan = AttentionPlan(pool, table, [n], [n], 8, query_dtype=query)
        assert torch.isfinite(attend(plan, 0, q)).all()
        pool._arrays[which][slot, :, :-4] = 0
        pool._arrays[which][slot, :, -4:] = 255
        got = attend(plan, 0, q)
        want, tol = reference(q[:-1], k[0], v[0], bs, table, [n - 1], [n - 1])
        assert ((got[:-1].double() - want).abs() <= tol).all()
        assert torch.isnan(got[-1]).all()


@pytest.mark.parametrize("kv_heads, dim", [(8, 128), (4, 96), (4, 64), (3, 72)])
@pytest.mark.parametrize("format", FORMATS)
def test_long_streams_beside_rows_that_are_no_numbers(gpu, kv_heads, dim, format):
    """Every row that no query sees holds such groups: before the windows, behind the contexts
    in their last blocks, in blocks of nobody. One visible V has one: it shows in its group of
    its own sequence's outputs and nowhere else."""
    from iekv.engine.attention import AttentionPlan, attend

    contexts, bs, blocks, window, sinks = [5003 + 37 * i for i in range(64)], 16, 400, 4000, 3
    pool, k, v = make_pool(blocks, bs, kv_heads, dim, format, BF16, 41)
    gen = torch.Generator().manual_seed(42)
    half = blocks // 2
    tables, seen = [], torch.zeros(blocks * bs, dtype=torch.bool)
    for c in contexts:                        # blocks of the window from one half of the pool,
        first, n = (c - window) // bs, -(-c // bs)      # hidden ones from the other
        table = torch.randint(half, (n,), generator=gen)
        table[1:first] += half
        table[0], table[-1] = 2 * half - 1, 2 * half - 2
        tables.append(table.tolist())
        for j in list(range(sinks)) + list(range(max(first, 1) * bs, c)):
            if j >= c - window or j < sinks:
                seen[int(table[j // bs]) * bs + j % bs] = True
    hidden = ~seen
    assert hidden.sum() > half * bs // 2
    for t in pool._arrays:
        t[hidden.cuda(), :, -4:] = 255
    q = queries_of(64, 4 * kv_heads, dim, BF16, 43)
    got, _ = check(q, k[0], v[0], pool, tables, contexts, [1] * 64, window=window, sinks=sinks)
    assert torch.isfinite(got).all()
    slot, shown = tables[9][0] * bs + 1, 1    # a sink of all sequences
    codes = 16 if format == "mxfp4" else 32
    pool._arrays[1][slot, kv_heads - 1, shown * codes:shown * codes + codes] = 0
    pool._arrays[1][slot, kv_heads - 1, -4 + shown] = 255
    plan = AttentionPlan(pool, tables, contexts, [1] * 64, 4 * kv_heads, window=window, sinks=sinks)
    bad = torch.isnan(attend(plan, 0, q))
    want = torch.zeros_like(bad)
    want[:, 4 * (kv_heads - 1):, 32 * shown:32 * shown + 32] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("query", TYPES, ids=str)
def test_magnitudes(gpu, query, format):
    """Scores far apart, rows of very different size, and rows of zeros."""
    def rows(x):
        gen = torch.Generator().manual_seed(3)
        size = torch.exp2(torch.randn((len(x), 1, 1), generator=gen) * 3)
        size[torch.rand((len(x), 1, 1), generator=gen) < 0.1] = 0
        return x * size

    contexts, queries = [150, 90], [1, 90]
    pool, k, v = make_pool(20, 16, 2, 64, format, query, 28, rows=rows)
    tables = make_tables(contexts, 16, 20, 29)
    q = queries_of(91, 8, 64, query, 30, scale=30.0)
    check(q, k[0], v[0], pool, tables, contexts, queries)
    check(q, k[0], v[0], pool, tables, contexts, queries, scale=-0.3)
    check(q, k[0], v[0], pool, tables, contexts, queries, scale=0.0)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("n", [1, 70])
def test_values_that_float16_does_not_hold(gpu, format, n):
    """float16 queries take a value past 65,504 as the infinity that reading it back in their
    type gives; one below its smallest as what it rounds to there."""
    from iekv.engine.attention import AttentionPlan, attend
    from iekv.engine.slots import gather_rows, write_slots

    pool, k, v = make_pool(8, 16, 2, 64, format, F16, 31)
    tables, context = make_tables([100], 16, 8, 32), 100
    rows = torch.randn((1, 2, 64), generator=torch.Generator().manual_seed(1)).cuda()
    rows[0, 0, 9] = 9.0e4
    rows[0, 1] *= 2.0 ** -20
    at = tables[0][40 // 16] * 16 + 40 % 16
    write_slots(pool, 0, torch.zeros_like(rows), rows, [at])
    q = queries_of(n, 8, 64, F16, 33)
    plan = AttentionPlan(pool, tables, [context], [n], 8, query_dtype=F16)
    got = attend(plan, 0, q)
    sees = torch.arange(context - n, context) >= 40
    assert torch.isinf(got[sees, :4, 9]).all() and torch.isfinite(got[~sees]).all()
    # Of the others the definition, over what is read back.
    k16, v16 = (gather_rows(pool, o, list(range(8)), 128, dtype=F16) for o in (0, 1))
    v16[at, 0, 9] = 0
    want, tol = reference(q, k16, v16, 16, tables, [context], [n])
    keep = torch.ones(64, dtype=torch.bool)
    keep[9] = False
    assert ((got.double() - want).abs() <= tol)[..., keep].all()


@pytest.mark.parametrize("format", FORMATS)
def test_strides_places_and_odd_addresses(gpu, format):
    from iekv.engine.attention import AttentionPlan, attend
    from iekv.engine.quantized import QuantizedPool

    contexts, queries = [70, 200], [5, 1]
    for query in (BF16, F32):
        pool, k, v = make_pool(20, 16, 2, 72, format, query, 34)
        tables = make_tables(contexts, 16, 20, 35)
        q = queries_of(6, 8, 72, query, 36)
        want, plan = check(q, k[0], v[0], pool, tables, contexts, queries)
        fused = torch.zeros((6, 8 * 72 + 100), dtype=query, device="cuda")
        fused[:, 1:577] = q.view(6, 576)
        assert torch.equal(attend(plan, 0, fused[:, 1:577].view(6, 8, 72)), want)
        assert torch.equal(attend(plan, 0, q.permute(1, 0, 2).contiguous().permute(1, 0, 2)), want)
        odd = []
        for t in pool._arrays:
            o = torch.zeros(t.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(t.shape)
            o.copy_(t)
            odd.append(o)
        other = AttentionPlan(QuantizedPool(odd[:1], odd[1:], 16, format), tables, contexts,
                              queries, 8, query_dtype=query)
        assert torch.equal(attend(other, 0, q), want)
        again = q.clone()
        assert attend(plan, 0, again, out=again) is again and torch.equal(again, want)


def test_offsets_past_32_bits(gpu):
    """A cache of more than 4 GiB: blocks at its end, for single tokens and a prompt."""
    from iekv.engine.quantized import QuantizedPool, allocate_quantized_pool
    from iekv.engine.slots import gather_rows, write_slots

    bs, kv_heads, dim, blocks = 16, 8, 128, 300_000
    k, v = allocate_quantized_pool(blocks, bs, 1, kv_heads, dim, format="mxint8")
    pool = QuantizedPool(k, v, bs, "mxint8")
    last = 80
    rows = torch.randn((2, last * bs, kv_heads, dim),
                       generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    write_slots(pool, 0, rows[0], rows[1],
                torch.arange((blocks - last) * bs, blocks * bs, device="cuda"))
    # The definition over the last blocks alone, by their place among these.
    contexts, queries = [500, 100], [1, 100]
    near = [[last - 1 - 2 * i for i in range(32)], [last - 2 - 2 * i for i in range(7)]]
    tables = [[b + blocks - last for b in t] for t in near]
    values = [gather_rows(pool, o, list(range(blocks - last, blocks)), last * bs) for o in (0, 1)]
    q = queries_of(101, 32, dim, BF16, 37)
    from iekv.engine.attention import AttentionPlan, attend

    got = attend(AttentionPlan(pool, tables, contexts, queries, 32), 0, q)
    want, tol = reference(q, *values, bs, near, contexts, queries)
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("format", FORMATS)
def test_a_step_writes_attends_and_is_replayed(gpu, format):
    """A decode step of three layers as a serving loop runs it: rows written, attention over
    them, in a captured graph, on another stream and eagerly."""
    from iekv.engine.attention import AttentionPlan, attend
    from iekv.engine.slots import gather_rows, write_slots

    contexts, queries, bs = [1500, 700, 33], [1, 1, 1], 16
    blocks = sum(-(-c // bs) for c in contexts) + 3
    pool, k, v = make_pool(blocks, bs, 2, 128, format, BF16, 38, layers=3)
    tables = make_tables(contexts, bs, blocks, 39)
    slots = torch.tensor([t[(c - 1) // bs] * bs + (c - 1) % bs
                          for t, c in zip(tables, contexts)], device="cuda")
    plan = AttentionPlan(pool, tables, contexts, queries, 8)
    new = torch.zeros((3, 2, 3, 2, 128), dtype=BF16, device="cuda")
    q = torch.zeros((3, 3, 8, 128), dtype=BF16, device="cuda")

    def step():
        outs = []
        for l in range(3):
            write_slots(pool, l, new[l, 0], new[l, 1], slots)
            outs.append(attend(plan, l, q[l]))
        return outs

    def fresh(seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        new.copy_(torch.randn(new.shape, generator=gen, device="cuda"))
        q.copy_(torch.randn(q.shape, generator=gen, device="cuda"))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(4):
        fresh(seed)
        graph.replay()
        replayed = [o.clone() for o in captured]
        eager = step()
        torch.cuda.synchronize()
        for l in range(3):
            assert torch.equal(replayed[l], eager[l])
            values = [gather_rows(pool, o, list(range(blocks)), blocks * bs)
                      for o in (l, 3 + l)]
            assert torch.equal(values[0][slots].cpu(),
                               decode(encode(new[l, 0], format), format).to(BF16))
            want, tol = reference(q[l], *values, bs, tables, contexts, queries)
            assert ((eager[l].double() - want).abs() <= tol).all()


def test_refusals(gpu):
    from iekv.engine.attention import AttentionPlan

    pool, k, v = make_pool(8, 16, 2, 64, "mxfp4", BF16, 40)
    args = ([[1, 2], [3]], [20, 5], [1, 5], 8)
    assert AttentionPlan(pool, *args).query_dtype == BF16
    with pytest.raises(ValueError, match="float64"):
        AttentionPlan(pool, *args, query_dtype=torch.float64)
    with pytest.raises(ValueError, match="float8"):
        AttentionPlan(pool, *args, query_dtype=torch.float8_e5m2)
    with pytest.raises(RuntimeError, match="type 4"):
        AttentionPlan(pool, *args, query_dtype=torch.float8_e4m3fn)
    with pytest.raises(IndexError, match="out of range"):
        AttentionPlan(pool, [[1, 8], [3]], *args[1:])


# contexts, queries, shared blocks, options: chunks alone, beside single tokens in one launch and
# behind long streams, in parts, and sequences that share their first blocks.
WEIGHTED = {
    "prompt": ([129], [129], 0, {}),
    "chunks": ([300, 200, 77, 640], [1, 131, 3, 333], 0, {}),
    "window": ([900], [500], 0, dict(window=170, sinks=9)),
    "parts": ([6000], [33], 0, {}),
    "shared": ([1300 + i for i in range(40)], [1] * 40, 80, {}),
}


@pytest.mark.parametrize("step", list(WEIGHTED))
@pytest.mark.parametrize("dim", [128, 72])
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("query", [BF16, F16], ids=str)
def test_weights_are_held_as_two_numbers(gpu, query, format, dim, step):
    """A weight is its value rounded to the queries' type and what that leaves, rounded: off by
    u^2 of it (u: half a step) where one number would be off by u. V of mixed signs, so that an
    output, whose own rounding is allowed u of it, is small beside A = sum p |v|; short queries,
    so that scores are nearly exact. Twice as many terms are summed in 32 bits."""
    from iekv.engine.attention import AttentionPlan, attend

    contexts, queries, shared, options = WEIGHTED[step]
    bs, kv_heads, group = 16, 2, 4
    blocks = sum(-(-c // bs) for c in contexts) + 3
    pool, k, v = make_pool(blocks, bs, kv_heads, dim, format, query, 71)
    tables = make_tables(contexts, bs, blocks, 72, shared)
    q = queries_of(sum(queries), kv_heads * group, dim, query, 73, scale=0.05)
    plan = AttentionPlan(pool, tables, contexts, queries, kv_heads * group, query_dtype=query,
                         shared_blocks=shared, **options)
    got = attend(plan, 0, q)
    want, tol = reference(q, k[0], v[0], bs, tables, contexts, queries, **options)
    a, _ = reference(q, k[0], v[0].abs(), bs, tables, contexts, queries, **options)
    u, n = torch.finfo(query).eps / 2, max(contexts)
    tol = tol + (u * u - u + n * 2.0 ** -24) * a
    if query == F16:                     # the end of float16 below weights held 2^7 above: check
        tol = tol + 2.0 ** -32 * n * v[0].double().abs().amax()
    off = (got.double() - want).abs()
    assert not torch.isnan(off).any()
    worst = (off / tol.clamp_min(1e-300)).max().item()   # a key of zeros alone: both are 0
    assert worst <= 1.0, f"{worst} times the tolerance"


# float16 numbers that a format rounds to float16's infinity, and the next below, which it does not.
ENDS = {"mxfp8": [(63488.0, 63456.0), (65504.0, 61440.0)],
        "mxint8": [(65056.0, 65024.0), (65504.0, 64992.0)],
        "mxfp4": [(57344.0, 57312.0), (65504.0, 49152.0)]}


@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("format", FORMATS)
def test_the_end_of_float16(gpu, format, rows):
    """Rows of float16 near its largest, as the documents have it: read back in float16 they are
    infinite from there on, finite below and in wider types; attention takes them as read."""
    from iekv.engine.attention import AttentionPlan, attend
    from iekv.engine.quantized import QuantizedPool, allocate_quantized_pool
    from iekv.engine.slots import gather_rows, write_slots

    context, dim = 80, 64
    for past, below in ENDS[format]:
        k, v = allocate_quantized_pool(5, 16, 1, 1, dim, format=format)
        pool = QuantizedPool(k, v, 16, format)
        gen = torch.Generator(device="cuda").manual_seed(81)
        key = torch.randn((context, 1, dim), generator=gen, device="cuda").half()
        value = torch.randn((context, 1, dim), generator=gen, device="cuda").half()
        value[3, 0, 5], value[3, 0, 40] = past, -below          # of a group of their own each
        table = list(range(5))
        write_slots(pool, 0, key, value, list(range(context)))
        read = gather_rows(pool, 1, table, context, dtype=F16)
        assert read[3, 0, 5] == float("inf")
        assert torch.isinf(read).sum() == 1 and not torch.isnan(read).any()
        wide = gather_rows(pool, 1, table, context, dtype=F32)
        assert torch.isfinite(wide).all() and wide[3, 0, 5] == 65536.0
        assert torch.equal(wide.half(), read)
        q = torch.randn((rows, 2, dim), generator=gen, device="cuda").half() * 0.1
        plan = AttentionPlan(pool, [table], [context], [rows], 2, query_dtype=F16)
        got = attend(plan, 0, q)
        if rows == 1 or context - rows >= 3:                    # every row sees the third key
            assert (got[..., 5] == float("inf")).all()
        assert torch.isfinite(got[..., :5]).all() and torch.isfinite(got[..., 6:]).all()
        wider = attend(AttentionPlan(pool, [table], [context], [rows], 2, query_dtype=F32), 0,
                       q.float())
        assert torch.isfinite(wider).all()
