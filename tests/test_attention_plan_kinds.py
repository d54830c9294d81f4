"""Steps of every kind that a plan can have, each cut so that every visible key is read once (CPU).

What a step takes whole and which prefixes it shares goes by sizes; here these limits vary, so
that steps small enough to be checked key by key are of every kind.
"""
from __future__ import annotations

import random
import subprocess

import pytest

from conftest import PACKAGE_ROOT, ROOT


@pytest.fixture(scope="module")
def checker(tmp_path_factory):
    out = tmp_path_factory.mktemp("plan") / "attention_plan_kinds_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=address,undefined",
                    "-I", str(PACKAGE_ROOT / "csrc"), "-I", str(ROOT / "tests"),
                    str(ROOT / "tests" / "attention_plan_kinds_check.cpp"), "-o", str(out)],
                   check=True)
    return out


def run(checker, cases):
    text = "".join(f"{' '.join(map(str, shape))} {len(seqs)} "
                   f"{' '.join(f'{c} {n}' for c, n in seqs)}\n" for shape, seqs in cases)
    out = subprocess.run([str(checker)], input=text, capture_output=True, text=True, check=True)
    lines = out.stdout.splitlines()
    assert len(lines) == len(cases)
    for case, line in zip(cases, lines):
        assert line.startswith("ok"), (case, line)
    return [set(line.split()[2:]) for line in lines]


ANY = 1 << 30       # bytes a key, so that any prefix of two sequences is worth sharing


def steps():
    # few_keys key_bytes group kv_heads block window sinks shared wide_rows units, (context, queries)
    rng = random.Random(12)
    for _ in range(500):
        block = rng.choice([1, 3, 8, 16])
        shared = block * rng.choice([0, 0, 1, 7, 60])
        seqs = []
        for _ in range(rng.randint(1, 7)):
            context = shared + rng.choice([0, 1, 3, 70, 400, 1500]) + rng.randint(0, 40)
            most = rng.choice([0, 1, 1, 2, 5, 40, 150])
            seqs.append((context, min(context, rng.randint(min(most, 1), most))))
        yield ((rng.choice([0, 64, 512, 1024]), rng.choice([1, 512, ANY, ANY]),
                rng.choice([1, 2, 4, 7, 20, 100]), rng.choice([1, 2, 2, 3, 4, 6, 8]), block,
                rng.choice([0, 0, 1, 9, 200, 1500]), rng.choice([0, 3, 70]), shared,
                rng.choice([128, 128, 64, 0]), rng.choice([1, 1, 8, 256])), seqs)


def test_steps_of_every_kind_read_every_visible_key_once(checker):
    found = {}
    for kinds in run(checker, list(steps())):
        for k in kinds:
            found[k] = found.get(k, 0) + 1
    for kind in ("shared", "mixed", "narrow-parts", "wide-parts", "streams", "together-1",
                 "together-2", "together-4"):
        assert found.get(kind, 0) >= 10, found


@pytest.mark.parametrize("window, sinks, shares", [
    (0, 0, True), (4000, 4, True), (1100, 4, True), (600, 4, False), (100, 4, False),
    (100, 2000, True), (1, 0, False)])
def test_prefixes_that_a_window_has_left_behind_are_not_shared(checker, window, sinks, shares):
    """96 sequences of 2,560 tokens behind 2,048: what of them the last tokens see counts."""
    shape = (1024, 512, 4, 8, 16, window, sinks, 2048, 128, 256)
    kinds, = run(checker, [(shape, [(2560, 1)] * 96)])
    assert ("shared" in kinds) == shares, kinds


@pytest.mark.parametrize("key_bytes, kv_heads, group, shared, contexts, shares", [
    (512, 8, 4, 16, [1200] * 96, False),             # one block of many sequences
    (512, 8, 4, 256, [1200] * 96, False),
    (512, 8, 4, 1024, [1200] * 96, True),
    (512, 8, 4, 512, [612] * 8, True),
    (512, 8, 4, 512, [612] * 4, False),              # too few sequences
    (256, 8, 8, 512, [612] * 64, False),             # 8-bit keys
    (256, 8, 8, 1024, [1124] * 64, True),
    (256, 8, 8, 14336, [14400] * 16, True),
    (256, 2, 7, 512, [662] * 24, False),
    (512, 2, 4, 2048, [2100] * 16, True),
    (512, 8, 4, 2048, [2100], False),                # alone
])
def test_prefixes_are_shared_where_that_saves_more_than_a_join(checker, key_bytes, kv_heads, group,
                                                               shared, contexts, shares):
    shape = (1024, key_bytes, group, kv_heads, 16, 0, 0, shared, 128, 256)
    kinds, = run(checker, [(shape, [(c, 1) for c in contexts])])
    assert ("shared" in kinds) == shares, kinds
