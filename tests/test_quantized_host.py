"""Microscaled caches: what the host decides and refuses (CPU)."""
from __future__ import annotations

import ctypes
import re
import subprocess

import pytest
import torch

from conftest import PACKAGE_ROOT, ROOT
from quantized_reference import CODES, FORMATS, decode, encode
from test_attention_plan import make, ops  # noqa: F401  (the library, and a plan of two sequences)
from test_ops_host import on_stub  # noqa: F401  (the library over a HIP that runs nothing)

INVALID, RANGE = -1, -4
MOST = (2 ** 32 - 1) // 256          # workgroups of a launch


def test_types_and_structure_agree_with_the_header():
    from iekv import _ops

    text = (ROOT / "include" / "iekv_ops.h").read_text()
    for name in ("MXFP8", "MXINT8", "MXFP4"):
        value = re.search(rf"IEKV_TYPE_{name} = (\d+)", text).group(1)
        assert int(value) == getattr(_ops, f"IEKV_TYPE_{name}")
    for name in ("INLINE_SLOTS", "INLINE_BLOCKS"):
        value = re.search(rf"#define IEKV_MX_{name} (\d+)", text).group(1)
        assert int(value) == getattr(_ops, f"MX_{name}")
    assert ctypes.sizeof(_ops.MxCache) == 24


def test_records(ops):  # noqa: F811
    from iekv.engine.quantized import FORMATS as TYPES
    from iekv.engine.quantized import record_bytes

    assert set(TYPES) == set(FORMATS)
    for format in FORMATS:
        for dim in range(8, 129, 8):
            size = dim // (2 if format == "mxfp4" else 1) + 4
            assert record_bytes(format, dim) == size == ops.iekv_mx_head_bytes(TYPES[format], dim)
        for dim in (0, -8, 4, 12, 136):
            with pytest.raises(ValueError, match=f"head_dim {dim}"):
                record_bytes(format, dim)
            assert ops.iekv_mx_head_bytes(TYPES[format], dim) == 0
    with pytest.raises(ValueError, match="no format 'fp8'"):
        record_bytes("fp8", 128)
    assert ops.iekv_mx_head_bytes(4, 128) == ops.iekv_mx_head_bytes(8, 128) == 0


def test_the_definition():
    """The oracle's own rounding: nearest, ties to even codes, nothing past the largest."""
    x = torch.zeros(1, 32, dtype=torch.float64)
    x[0, :9] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.26])
    assert decode(encode(x, "mxfp4"), "mxfp4")[0, :9].tolist() == \
        [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -0.5]
    x[0, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5])
    assert decode(encode(x, "mxint8"), "mxint8")[0, :4].tolist() == [127.0, 0.0, 2.0, -2.0]
    x[0, :4] = torch.tensor([448.0, 17.0, 19.0, -2.0 ** -10])
    assert decode(encode(x, "mxfp8"), "mxfp8")[0, :4].tolist() == [448.0, 16.0, 20.0, 0.0]
    gen = torch.Generator().manual_seed(1)
    for format in FORMATS:
        rows = torch.randn((50, 3, 80), generator=gen, dtype=torch.float64)
        rows *= torch.exp2(torch.randn((50, 3, 1), generator=gen) * 12)
        got = decode(encode(rows, format), format)
        # By brute force over every code of a group's own exponent and of one less: its largest
        # is within the type's, and would not be there.
        scale = torch.ldexp(torch.ones((), dtype=torch.float64),
                            encode(rows, format)[..., -4:].int() - 127)
        top = {"mxfp8": 448.0, "mxint8": 127.0, "mxfp4": 6.0}[format]
        values = CODES[format][torch.isfinite(CODES[format])]
        values = values[values.abs() <= top]
        for g in range(3):
            part, s = rows[..., g * 32:g * 32 + 32], scale[..., g:g + 1]
            assert (part.abs().amax(-1) <= top * s[..., 0]).all()
            assert (part.abs().amax(-1) > top / 2 * s[..., 0]).all()
            off = (part[..., None] - values * s[..., None]).abs().amin(-1)
            assert torch.equal((part - got[..., g * 32:g * 32 + 32]).abs(), off)


@pytest.mark.parametrize("format, of_value, of_largest, smallest", [
    ("mxfp8", 2.0 ** -4, 2.0 ** -17, 2.0 ** -110), ("mxint8", 0.0, 1 / 127, 2.0 ** -101),
    ("mxfp4", 2.0 ** -2, 1 / 12, 2.0 ** -102)])
def test_how_far_an_element_is_off(format, of_value, of_largest, smallest):
    """As the module says: a part of the value, or of its group's largest where that is more, or
    half a step of the least power. Groups whose largest is just past what the power before would
    hold, and elements between two codes there, are where the bounds are met."""
    top = {"mxfp8": 448.0, "mxint8": 127.0, "mxfp4": 6.0}[format]
    gen = torch.Generator().manual_seed(5)
    groups = torch.randn((4000, 32), generator=gen, dtype=torch.float64)
    groups *= torch.exp2(torch.randn((4000, 32), generator=gen, dtype=torch.float64) * 6)
    values = CODES[format][torch.isfinite(CODES[format])].unique()
    halves = (values[1:] + values[:-1]) / 2
    edges = torch.zeros((len(halves), 32), dtype=torch.float64)
    edges[:, 0] = top / 2 * (1 + 2.0 ** -30)                  # of steps of 1: not held in halves
    edges[:, 1] = halves * (1 - 2.0 ** -40)
    edges[:, 2] = -halves * (1 + 2.0 ** -40)
    edges = edges[edges.abs().amax(-1) == edges[:, 0]]
    tiny = torch.cat((groups, edges)) * 2.0 ** -105
    held = torch.cat((groups, edges, edges * 2.0 ** -60, edges * 2.0 ** 60))
    for x, least in ((held, 0.0), (tiny, smallest)):
        off = (x - decode(encode(x, format), format)).abs()
        bound = torch.maximum(of_value * x.abs(), of_largest * x.abs().amax(-1, keepdim=True))
        assert (off <= bound.clamp(min=least)).all()
    # And no smaller ones hold: mxint8's is past 2^-7, e4m3's small ones are lost altogether.
    off = (edges - decode(encode(edges, format), format)).abs()
    relative = off / edges.abs().amax(-1, keepdim=True)
    if of_value:
        assert (off[:, 1] / edges[:, 1].abs()).nan_to_num(0.0).max() > of_value
        assert relative[:, 1:].max() > of_largest
        assert ((off == edges.abs()) & (edges != 0)).any()
    else:
        assert relative.max() > 0.999 * of_largest > 2.0 ** -7


def test_pools_of_host_tensors_are_refused():
    from iekv.engine.quantized import QuantizedPool, allocate_quantized_pool

    k, v = allocate_quantized_pool(4, 8, 2, 2, 32, format="mxfp8", device="cpu")
    assert len(k) == len(v) == 2 and k[0].shape == (32, 2, 36) and k[0].dtype == torch.uint8
    with pytest.raises(ValueError, match="GPU"):
        QuantizedPool(k, v, 8, "mxfp8")
    with pytest.raises(ValueError, match="no format"):
        QuantizedPool(k, v, 8, "int8")


@pytest.mark.parametrize("cache_type, query_type, taken", [
    *[(c, q, True) for c in (5, 6, 7) for q in (1, 2, 3)], (8, 3, False), (8, 1, False),
    (5, 4, False), (7, 5, False), (6, 0, False)])
def test_plans_take_microscaled_caches(ops, cache_type, query_type, taken):  # noqa: F811
    rc, out, message = make(ops, cache_type=cache_type, query_type=query_type)
    assert (rc == 0) == taken
    if taken:
        ops.iekv_attention_plan_destroy(out)
    else:
        assert rc == INVALID and f"cache of type {cache_type}" in message


def test_wide_items_that_all_run_at_once_pair_long_with_short(ops):  # noqa: F811
    """512 workgroups, two to a compute unit: item i runs beside item i + 32."""
    n, context = 2048, 7777
    blocks = -(-context // 16)
    rc, plan, _ = make(ops, contexts=(context,), queries=(n,), tables=(tuple(range(blocks)),),
                       num_blocks=blocks, num_heads=32, num_kv_heads=8, head_dim=128)
    assert rc == 0
    words, count = ctypes.POINTER(ctypes.c_int32)(), ctypes.c_int64()
    tokens, workspace = ctypes.c_int64(), ctypes.c_int64()
    ops.iekv_attention_plan_info(plan, ctypes.byref(words), ctypes.byref(count),
                                 ctypes.byref(tokens), ctypes.byref(workspace))
    items = [words[12 * i:12 * i + 12] for i in range(64)]
    keys = [it[4] - it[3] + it[6] - it[5] for it in items]
    assert sorted(keys) == [context - n + 32 * (i + 1) for i in range(64)]
    assert keys[:32] == sorted(keys, reverse=True)[:32]
    pairs = [a + b for a, b in zip(keys[:32], keys[32:])]
    assert max(pairs) - min(pairs) <= 32
    ops.iekv_attention_plan_destroy(plan)


@pytest.mark.parametrize("cache_type, parts", [(3, 64), (4, 64), (5, 32), (6, 32), (7, 32)])
def test_few_sequences_are_cut_into_a_workgroup_for_each_compute_unit(ops, cache_type, parts):  # noqa: F811
    """Of microscaled caches; of the others two."""
    context, blocks = 16384, 1024
    rc, plan, _ = make(ops, contexts=(context,), queries=(1,), tables=(tuple(range(blocks)),),
                       num_blocks=blocks, num_heads=64, num_kv_heads=8, head_dim=128,
                       cache_type=cache_type)
    assert rc == 0
    words, count = ctypes.POINTER(ctypes.c_int32)(), ctypes.c_int64()
    tokens, workspace = ctypes.c_int64(), ctypes.c_int64()
    ops.iekv_attention_plan_info(plan, ctypes.byref(words), ctypes.byref(count),
                                 ctypes.byref(tokens), ctypes.byref(workspace))
    items = [words[12 * i:12 * i + 12] for i in range(parts)]
    assert all(it[:2] == [0, 1] and it[8:10] == [context - 1] * 2 for it in items)
    assert sum(it[4] - it[3] + it[6] - it[5] for it in items) == context
    ops.iekv_attention_plan_destroy(plan)


PARTS = r"""
#include <cstdio>
#include <map>
#include "attention_plan.h"
using namespace iekv_attention;

int main() {
  int turned = 0;
  for (int units = 16; units <= 256; units += 16)
    for (int heads = 1; heads <= 4; ++heads)
      for (int many = 8; many <= 56; many += 8) {
        const int context = 2400 + 8 * many;
        std::vector<Sequence> seqs{{context, 0, 0, 0}, {context - 900, 0, 0, 200}};
        int tokens = 0;
        for (Sequence& s : seqs) s.token0 = tokens, s.queries = many, tokens += many;
        const Plan p = make_plan(Shape{4, heads, 16, 0, 0, 0, 128}, seqs, units);
        std::map<int, const Item*> of;               // by slot
        bool in_order = true;
        for (int i = 0; i < p.wide.n; ++i) {
          const Item& it = p.items[p.wide.first + i];
          in_order = in_order && (!i || keys_of(it) <= keys_of((&it)[-1]));
          for (int t = 0; t < it.tokens && it.slot >= 0; ++t) of[it.slot + 4 * t] = &it;
        }
        turned += !in_order && !p.join_parts.empty();
        for (size_t e = 0; e < p.join_tokens.size(); ++e)
          for (int i = p.join_starts[e] + 1; i < p.join_starts[e + 1]; ++i) {
            const Item &x = *of.at(p.join_parts[i - 1]), &y = *of.at(p.join_parts[i]);
            if (keys_of(x) < keys_of(y) || (keys_of(x) == keys_of(y) && x.a0 + x.b0 >= y.a0 + y.b0))
              return std::printf("%d units, %d heads, %d tokens\n", units, heads, many), 1;
          }
      }
  std::printf("%d\n", turned);
}
"""


def test_parts_are_joined_in_one_order(tmp_path):
    """The longest first, then by their keys, however the items that make them are ordered."""
    (tmp_path / "parts.cpp").write_text(PARTS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I",
                    str(PACKAGE_ROOT / "csrc"), str(tmp_path / "parts.cpp"), "-o",
                    str(tmp_path / "parts")], check=True)
    run = subprocess.run([str(tmp_path / "parts")], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout
    assert int(run.stdout) > 0                       # of steps whose items are in another order


CALLS = """
def cache(**over):
    fields = dict(dict(cache_type=5, num_kv_heads=8, head_dim=128, block_size=16, num_blocks=100),
                  **over)
    return ctypes.byref(_ops.MxCache(**fields))

def u64(*x):
    return (ctypes.c_uint64 * len(x))(*x)

def i64(*x):
    return (ctypes.c_int64 * len(x))(*x)

def write(k=u64(1 << 20), v=u64(1 << 21), layers=1, row=3, n=5, rows=1 << 22, slots=1 << 23,
          strides=i64(5120, 1024, 128), **over):
    return ops.iekv_mx_write_slots(cache(**over), k, v, layers, row, rows, strides, rows, strides,
                                   slots, n, 77)

def read(arrays=u64(1 << 20), n=1, table=1 << 21, context=20, out_type=3, out=1 << 22, **over):
    return ops.iekv_mx_read_rows(cache(**over), arrays, n, table, context, out_type, out, 77)

def said(rc):
    return [rc, ops.iekv_ops_last_error().decode() if rc else ""]
"""

SHAPES = [("cache_type=4", "4 is no microscaled type"), ("cache_type=8", "8 is no microscaled"),
          ("num_kv_heads=0", "num_kv_heads 0"), ("num_kv_heads=4097", "num_kv_heads 4097"),
          ("head_dim=0", "head_dim 0"), ("head_dim=12", "head_dim 12"),
          ("head_dim=136", "head_dim 136"), ("block_size=0", "block_size 0"),
          ("num_blocks=0", "num_blocks 0"), ("num_blocks=1 << 31", "num_blocks 2147483648")]


def test_refusals_come_before_anything_is_enqueued(on_stub):  # noqa: F811
    cases = [(f"{f}({a})", want) for f in ("write", "read") for a, want in SHAPES]
    cases += [("write(row=4)", "rows of type 4"), ("write(row=0)", "rows of type 0"),
              ("write(layers=-1)", "-1 layers"), ("write(n=-1)", "of -1 tokens"),
              *[(f"write({a}=None)", "null") for a in ("k", "v", "rows", "slots", "strides")],
              ("read(out_type=5)", "values of type 5"), ("read(n=-2)", "-2 arrays"),
              ("read(context=-1)", "context of -1"),
              ("read(context=(1 << 30) + 1)", "context of 1073741825"),
              ("read(block_size=1 << 20, num_kv_heads=4096)", "too large"),
              *[(f"read({a}=None)", "null") for a in ("arrays", "table", "out")]]
    got = on_stub(CALLS + f"""
bad = [said(eval(call)) for call in {[c for c, _ in cases]!r}]
for f, x in ((ops.iekv_mx_write_slots_ids, i64(0, 1600)), (ops.iekv_mx_write_slots_ids, i64(-1))):
    bad.append(said(f(cache(), u64(1 << 20), u64(1 << 21), 1, 3, 1 << 22, i64(1, 1, 1), 1 << 22,
                      i64(1, 1, 1), x, len(x), 77)))
for x in ((0, 100), (7, -5)):
    bad.append(said(ops.iekv_mx_read_rows_ids(cache(), u64(1 << 20), 1,
                                              (ctypes.c_int32 * 2)(*x), 20, 3, 1 << 22, 77)))
bad.append(said(ops.iekv_mx_write_slots(None, *[None] * 2, 0, 3, *[None] * 5, 0, None)))
bad.append(said(ops.iekv_mx_read_rows(None, None, 0, None, 0, 3, None, None)))
none = [write(n=0, k=None, rows=None), write(layers=0, v=None), read(context=0, out=None),
        read(n=0, arrays=None)]
print(json.dumps([bad, none, launches()]))
""")
    ids = [("", "slot 1600 out of range"), ("", "slot -1 out"), ("", "block id 100 out of range"),
           ("", "block id -5 out")]
    last = [("", "cache is null")] * 2
    assert len(got[0]) == len(cases + ids + last)
    for (rc, message), (call, want) in zip(got[0], cases + ids + last):
        assert rc == (RANGE if (call, want) in ids else INVALID) and want in message, (call, rc)
    assert got[1] == [0, 0, 0, 0] and got[2] == []


def test_arrays_at_even_distances_share_a_launch(on_stub):  # noqa: F811
    """All layers of a pool in one launch; of arrays in no order as many as lie so."""
    got = on_stub(CALLS + """
even = u64(*[(1 << 30) + 4096 * i for i in range(40)])
odd = u64(*[(1 << 30) + 4096 * i for i in (0, 1, 2, 7, 9, 10, 5)])
stub.hipSetDevice(3)
rcs = [write(k=even, v=even, layers=40), write(k=even, v=odd, layers=7), write(layers=1),
       read(arrays=odd, n=7), read(arrays=even, n=40)]
print(json.dumps([rcs, launches()]))
""")
    assert got[0] == [0] * 5
    grids = [x[1:4] for x in got[1]]
    assert {x[0] for x in got[1]} == {3} and {x[4] for x in got[1]} == {77}
    # Two layers or arrays a workgroup.
    assert [x[1] for x in grids] == [20, 2, 1, 1, 1, 2, 1, 1, 20]


def test_steps_of_any_size_run_in_several_launches(on_stub):  # noqa: F811
    got = on_stub(CALLS + """
rc = write(n=(1 << 28) + 5, num_kv_heads=16)
print(json.dumps([said(rc), launches()]))
""")
    assert got[0][0] == 0, got[0]
    lanes = 16 * 16                                  # of a token
    assert len(got[1]) > 1 and all(x[1] <= MOST for x in got[1])
    assert sum(x[1] for x in got[1]) == ((1 << 28) + 5) * lanes // 256
    got = on_stub(CALLS + """
rcs = [read(context=(1 << 30) - 5), read(context=(1 << 29) + 1, block_size=1000, out_type=1)]
slots = list(range(300)) + [7]
rcs.append(ops.iekv_mx_write_slots_ids(cache(), u64(1 << 20), u64(1 << 21), 1, 3, 1 << 22,
                                       i64(1, 1, 1), 1 << 22, i64(1, 1, 1), i64(*slots), 301, 77))
ids = (ctypes.c_int32 * 600)(*([5] * 600))
rcs.append(ops.iekv_mx_read_rows_ids(cache(), u64(1 << 20), 1, ids, 9591, 3, 1 << 22, 77))
print(json.dumps([rcs, launches()]))
""")
    assert got[0] == [0] * 4
    grids = [x[1] for x in got[1]]
    assert max(grids) <= MOST
    rows = [grids.pop() for _ in range(6)][::-1]     # the lists' launches: 128 slots, 256 blocks
    assert rows[:3] == [128 // 2, 128 // 2, -(-45 // 2)]
    assert rows[3:] == [4096 // 2, 4096 // 2, -(-(9591 - 8192) // 2)]
    first = 1 + (((1 << 30) - 5) * 128 - 1) // 256   # of bf16: 16 lanes a head, 8 heads
    assert abs(sum(grids) - first - ((1 << 29) + 1)) <= len(grids)


@pytest.mark.parametrize("cache_type, dim, at_once", [
    (5, 128, 2), (5, 96, 2), (5, 64, 3), (6, 128, 2), (6, 96, 3), (6, 64, 3), (7, 128, 3),
    (7, 96, 3)])
def test_long_streams_are_cut_by_the_work_of_their_records(ops, cache_type, dim, at_once):  # noqa: F811
    """Into two or three workgroups of four heads for each of 256 compute units."""
    n, context = 48, 6000
    blocks = context // 16
    rc, plan, _ = make(ops, contexts=(context,) * n, queries=(1,) * n,
                       tables=(tuple(range(blocks)),) * n, num_blocks=blocks, num_heads=32,
                       num_kv_heads=8, head_dim=dim, cache_type=cache_type)
    assert rc == 0
    words, count = ctypes.POINTER(ctypes.c_int32)(), ctypes.c_int64()
    tokens, workspace = ctypes.c_int64(), ctypes.c_int64()
    ops.iekv_attention_plan_info(plan, ctypes.byref(words), ctypes.byref(count),
                                 ctypes.byref(tokens), ctypes.byref(workspace))
    items, keys = 0, 0
    while keys < n * context:
        it = words[12 * items:12 * items + 12]
        items, keys = items + 1, keys + it[4] - it[3] + it[6] - it[5]
    assert (at_once - 1) * 256 < items * 2 <= at_once * 256
    ops.iekv_attention_plan_destroy(plan)
