"""How a step's attention is cut into work items, and what the operators' C-ABI refuses (CPU)."""
from __future__ import annotations

import ctypes
import random
import re
import subprocess

import pytest

from conftest import PACKAGE_ROOT, ROOT

HEADER = ROOT / "include" / "iekv_ops.h"


@pytest.fixture(scope="module")
def ops():
    from iekv import _ops

    if not _ops.library_path().exists():
        pytest.fail(f"{_ops.library_path()} is not built (run __graft_entry__.build())")
    return _ops.lib()


@pytest.fixture(scope="module")
def checker(tmp_path_factory):
    out = tmp_path_factory.mktemp("plan") / "attention_plan_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=address,undefined",
                    "-I", str(PACKAGE_ROOT / "csrc"),
                    str(ROOT / "tests" / "attention_plan_check.cpp"), "-o", str(out)], check=True)
    return out


def steps():
    # group kv_heads block window sinks shared wide_rows units, (context, queries) ...
    yield (4, 8, 16, 0, 0, 0, 128, 256), [(1, 1)]
    yield (4, 8, 16, 0, 0, 0, 128, 256), [(0, 0), (7, 7), (5, 0), (1, 1)]
    yield (1, 4, 16, 128, 4, 0, 128, 256), [(270, 1)]
    yield (4, 8, 16, 64, 4, 0, 128, 256), [(777, 777)]
    yield (7, 2, 256, 1, 0, 0, 128, 256), [(300, 40), (20, 20)]
    yield (8, 8, 16, 5000, 100, 0, 128, 256), [(3000, 1), (2999, 3)]
    yield (8, 1, 16, 3, 600, 0, 128, 4), [(500, 30)]
    yield (4, 2, 16, 0, 0, 64, 128, 256), [(65, 1), (100, 36), (64, 1)]
    yield (4, 2, 16, 0, 0, 64, 128, 256), [(64, 40), (90, 50)]       # queries inside the prefix
    yield (3, 2, 8, 20, 5, 48, 128, 256), [(49, 1), (80, 10), (130, 3)]
    yield (128, 1, 16, 0, 0, 32, 128, 8), [(40, 3), (33, 1)]
    yield (2, 1, 16, 10, 2, 0, 0, 8), [(40, 30)]
    rng = random.Random(11)
    for _ in range(150):
        shared = rng.choice([0, 0, 8, 160])
        seqs = [(c, rng.randint(0, min(c, rng.choice([1, 5, 300]))))
                for c in (rng.randint(shared, shared + rng.choice([3, 40, 700]))
                          for _ in range(rng.randint(1, 6)))]
        yield ((rng.choice([1, 2, 3, 7, 8, 20, 100]), rng.randint(1, 8), 8,
                rng.choice([0, 0, 1, 9, 200]), rng.choice([0, 3, 70]), shared,
                rng.choice([128, 128, 64]), rng.choice([1, 64, 256])), seqs)


def test_every_visible_key_is_read_once(checker):
    cases = list(steps())
    text = "".join(f"{' '.join(map(str, shape))} {len(seqs)} "
                   f"{' '.join(f'{c} {n}' for c, n in seqs)}\n" for shape, seqs in cases)
    out = subprocess.run([str(checker)], input=text, capture_output=True, text=True, check=True)
    lines = out.stdout.splitlines()
    assert len(lines) == len(cases)
    for case, line in zip(cases, lines):
        assert line.startswith("ok"), (case, line)


def test_every_declared_operator_is_exported_and_bound(ops):
    from iekv import _ops

    names = set(re.findall(r"^\s*(?:int|int64_t|const char\*)\s+(iekv_\w+)\s*\(",
                           HEADER.read_text(), re.M))
    assert names == set(_ops.SIGNATURES)
    for name in names:
        assert hasattr(ops, name), name
    defined = dict(re.findall(r"#define (IEKV_\w+) ([^/\n]+)", HEADER.read_text()))
    assert ops.iekv_ops_abi_version() == _ops.ABI_VERSION == int(defined["IEKV_OPS_ABI_VERSION"])
    assert _ops.ATTENTION_MAX_DIM == int(defined["IEKV_ATTENTION_MAX_DIM"])
    assert _ops.ATTENTION_MAX_GROUP == int(defined["IEKV_ATTENTION_MAX_GROUP"])
    assert _ops.LOGPROBS_MAX_TOP == int(defined["IEKV_LOGPROBS_MAX_TOP"])


SHAPE = dict(num_heads=8, num_kv_heads=2, head_dim=64, block_size=16, num_blocks=10,
             query_type=3, cache_type=3, window=0, sinks=0, shared_blocks=0)


def make(ops, contexts=(20, 5), queries=(1, 5), tables=((1, 2), (3,)), **changes):
    from iekv import _ops

    flat = [b for t in tables for b in t]
    starts = [0]
    for t in tables:
        starts.append(starts[-1] + len(t))
    out = ctypes.c_void_p()
    rc = ops.iekv_attention_plan_create(
        ctypes.byref(_ops.AttentionShape(**dict(SHAPE, **changes))), len(contexts),
        (ctypes.c_int32 * len(contexts))(*contexts), (ctypes.c_int32 * len(queries))(*queries),
        (ctypes.c_int32 * max(1, len(flat)))(*flat), (ctypes.c_int64 * len(starts))(*starts),
        ctypes.byref(out))
    return rc, out, ops.iekv_ops_last_error().decode()


@pytest.mark.parametrize("changes, code, said", [
    (dict(num_kv_heads=0), -1, "num_kv_heads 0"),
    (dict(num_heads=7), -1, "7 query heads for 2 KV heads"),
    (dict(num_heads=258), -1, "129 query heads per KV head"),
    (dict(head_dim=136), -1, "head_dim 136"),
    (dict(head_dim=12), -1, "head_dim 12"),
    (dict(head_dim=0), -1, "head_dim 0"),
    (dict(block_size=0), -1, "block_size 0"),
    (dict(num_blocks=0), -1, "num_blocks 0"),
    (dict(query_type=4), -1, "type 4"),
    (dict(query_type=2), -1, "queries of type 2 on a cache of type 3"),
    (dict(cache_type=1), -1, "cache of type 1"),
    (dict(window=-1), -1, "window -1"),
    (dict(sinks=-2), -1, "sinks -2"),
    (dict(shared_blocks=-1), -1, "shared_blocks -1"),
    (dict(shared_blocks=1), -5, "sequence 1: a context of 5 does not fill 1 shared blocks"),
    (dict(shared_blocks=1, contexts=(20, 16)), -5, "sequence 1 does not begin with"),
    (dict(contexts=(33, 5)), -4, "context of 33 needs 3 blocks, table has 2"),
    (dict(tables=((1, 10), (3,))), -4, "block id 10 out of range for a pool of 10"),
    (dict(tables=((1, -1), (3,))), -4, "block id -1"),
    (dict(queries=(21, 5)), -1, "21 queries in a context of 20"),
    (dict(queries=(-1, 5)), -1, "-1 queries"),
    (dict(contexts=(-4, 5)), -1, "context of -4"),
    (dict(contexts=((1 << 30) + 1, 5)), -1, "context of 1073741825"),
])
def test_plans_refuse(ops, changes, code, said):
    rc, out, message = make(ops, **changes)
    assert rc == code and said in message, (rc, message)
    assert not out.value


def test_plans_hold_the_step(ops):
    rc, out, _ = make(ops, contexts=(20, 0, 5), queries=(1, 0, 5), tables=((1, 2, -1), (), (3,)))
    assert rc == 0
    words, n = ctypes.POINTER(ctypes.c_int32)(), ctypes.c_int64()
    tokens, workspace = ctypes.c_int64(), ctypes.c_int64()
    assert ops.iekv_attention_plan_info(out, ctypes.byref(words), ctypes.byref(n),
                                        ctypes.byref(tokens), ctypes.byref(workspace)) == 0
    assert tokens.value == 6 and n.value > 6
    assert words[n.value - 3:n.value] == [1, 2, 3]       # used table entries come last
    # Refusals of the call that enqueues come before any HIP call.
    args = [ctypes.c_void_p(64 * i) for i in range(1, 5)]
    assert ops.iekv_attend(out, None, *args[1:], 512, 64, 1.0, args[0], None, 0, None) == -1
    assert ops.iekv_attend(None, *args, 512, 64, 1.0, args[0], None, 0, None) == -1
    assert ops.iekv_attend(out, 68, *args[1:], 512, 64, 1.0, args[0], None, 0, None) == -1
    assert ops.iekv_attend(out, *args, 512, 64, float("nan"), args[0], None, 0, None) == -1
    assert ops.iekv_attention_plan_destroy(out) == 0
    rc, out, _ = make(ops, contexts=(), queries=(), tables=())
    assert rc == 0
    assert ops.iekv_attend(out, None, None, None, None, 0, 0, 1.0, None, None, 0, None) == 0
    ops.iekv_attention_plan_destroy(out)
    assert ops.iekv_attention_plan_destroy(None) == 0
    assert ops.iekv_attention_plan_create(None, 0, None, None, None, None, None) == -1


def test_split_steps_need_a_workspace(ops):
    tables = (tuple(range(1000)),)
    rc, out, _ = make(ops, contexts=(16000,), queries=(1,), tables=tables, num_blocks=1000)
    assert rc == 0
    words, n = ctypes.POINTER(ctypes.c_int32)(), ctypes.c_int64()
    tokens, workspace = ctypes.c_int64(), ctypes.c_int64()
    ops.iekv_attention_plan_info(out, ctypes.byref(words), ctypes.byref(n), ctypes.byref(tokens),
                                 ctypes.byref(workspace))
    assert workspace.value > 0
    args = [ctypes.c_void_p(64 * i) for i in range(1, 5)]
    for space, size in ((None, 0), (64, workspace.value - 1)):
        assert ops.iekv_attend(out, *args, 512, 64, 1.0, args[0], space, size, None) == -3
    assert ops.iekv_attend(out, *args, 512, 64, 1.0, args[0], 72, workspace.value, None) == -1
    ops.iekv_attention_plan_destroy(out)


@pytest.mark.parametrize("changes, code, said", [
    (dict(n_rows=-1), -1, "n_rows -1"),
    (dict(vocab=0), -1, "vocab 0"),
    (dict(vocab=1 << 31), -1, "vocab 2147483648"),
    (dict(top=65, vocab=1000), -1, "top 65"),
    (dict(top=-1), -1, "top -1"),
    (dict(top=8, vocab=7), -1, "top 8"),
    (dict(stride=-1), -1, "row_stride -1"),
    (dict(kind=4), -1, "type 4"),
    (dict(kind=0), -1, "type 0"),
    (dict(logits=None), -1, "null"),
    (dict(tokens=None), -1, "null"),
    (dict(ids=None), -1, "null"),
])
def test_logprobs_refuse(ops, changes, code, said):
    a = dict(dict(kind=1, logits=64, stride=100, n_rows=2, vocab=100, tokens=64, top=3,
                  logprobs=64, entropy=64, tops=64, ids=64), **changes)
    rc = ops.iekv_logprobs(a["kind"], a["logits"], a["stride"], a["n_rows"], a["vocab"],
                           a["tokens"], a["top"], a["logprobs"], a["entropy"], a["tops"], a["ids"],
                           None, 0, None)
    assert rc == code and said in ops.iekv_ops_last_error().decode()


def test_logprobs_of_no_rows(ops):
    assert ops.iekv_logprobs(1, None, 10, 0, 10, None, 0, None, None, None, None, None, 0,
                             None) == 0


def test_common_blocks():
    from iekv.engine.attention import common_blocks

    assert common_blocks([[1, 2, 3], [1, 2, 4]], [48, 40], 16) == 2
    assert common_blocks([[1, 2, 3], [1, 2, 3]], [48, 40], 16) == 2      # the third is not full
    assert common_blocks([[1, 2], [3, 2]], [32, 32], 16) == 0
    assert common_blocks([[1, 2]], [32], 16) == 0
    assert common_blocks([], [], 16) == 0
