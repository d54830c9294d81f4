"""What the operators' library decides on the host (CPU)."""
from __future__ import annotations

import json
import subprocess
import sys

import pytest
import torch

from conftest import PACKAGE_ROOT, ROOT
from test_attention_plan import make, ops  # noqa: F401  (the library, and a plan of two sequences)

INVALID = -1


@pytest.mark.parametrize("q, out, strides", [
    (1 << 20, (1 << 20) + 64, (512, 64)),          # some bytes further on
    ((1 << 20) + 16, 1 << 20, (512, 64)),
    (1 << 20, (1 << 20) + 6 * 1024 - 2, (512, 64)),    # the last element alone
    (1 << 20, 1 << 20, (64, 384)),                 # the same bytes in another order
    (1 << 20, 1 << 20, (1024, 64)),                # rows that lie further apart
    (1 << 20, 1 << 20, (0, 64)),                   # one row for all
    (1 << 20, (1 << 20) - 2048, (-512, 64)),       # rows that go back
])
def test_outputs_over_other_queries_are_refused(ops, q, out, strides):  # noqa: F811
    rc, plan, _ = make(ops)                        # 6 tokens of 8 heads of 64, 16 bits
    assert rc == 0
    assert ops.iekv_attend(plan, 64, 128, 192, q, *strides, 1.0, out, None, 0, None) == INVALID
    assert "overlaps" in ops.iekv_ops_last_error().decode()
    ops.iekv_attention_plan_destroy(plan)


# Run in a process of its own, without torch: the library over a HIP that runs nothing.
PRELUDE = """
import ctypes, json, sys
sys.path.insert(0, {package!r})
stub = ctypes.CDLL({stub!r}, mode=ctypes.RTLD_GLOBAL)
from iekv import _ops
ops = ctypes.CDLL(str(_ops.library_path()))
for name, (restype, argtypes) in _ops.SIGNATURES.items():
    getattr(ops, name).restype, getattr(ops, name).argtypes = restype, argtypes

def launches():
    out, row = [], (ctypes.c_int64 * 5)()
    for i in range(stub.stub_launches()):
        stub.stub_launch(i, row)
        out.append(list(row))
    return out

def device():
    d = ctypes.c_int()
    stub.hipGetDevice(ctypes.byref(d))
    return d.value

def plan(contexts, queries, bs=16, shared=0, **shape):
    counts = [-(-c // bs) for c in contexts]
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    flat = [b for n in counts for b in range(n)]
    fields = dict(dict(num_heads=8, num_kv_heads=2, head_dim=64, block_size=bs,
                       num_blocks=max(counts) + 1, query_type=3, cache_type=3,
                       shared_blocks=shared), **shape)
    out = ctypes.c_void_p()
    rc = ops.iekv_attention_plan_create(
        ctypes.byref(_ops.AttentionShape(**fields)), len(contexts),
        (ctypes.c_int32 * len(contexts))(*contexts), (ctypes.c_int32 * len(queries))(*queries),
        (ctypes.c_int32 * len(flat))(*flat), (ctypes.c_int64 * len(starts))(*starts),
        ctypes.byref(out))
    assert rc == 0, (rc, ops.iekv_ops_last_error())
    return out

def attend(p, stream=77):
    A = 1 << 44
    return ops.iekv_attend(p, A, 2 * A, 3 * A, 4 * A, 512, 64, 1.0, 5 * A, 6 * A, A, stream)
"""


@pytest.fixture(scope="module")
def on_stub(ops, tmp_path_factory):  # noqa: F811
    stub = tmp_path_factory.mktemp("stub") / "hip_stub.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC",
                    str(ROOT / "tests" / "hip_stub.cpp"), "-o", str(stub)], check=True)
    prelude = PRELUDE.format(package=str(PACKAGE_ROOT), stub=str(stub))

    def run(code):
        out = subprocess.run([sys.executable, "-c", prelude + code], capture_output=True,
                             text=True, timeout=120)
        assert out.returncode == 0, out.stderr[-2000:]
        return json.loads(out.stdout)

    return run


def test_attend_runs_on_the_device_its_plan_was_made_on(on_stub):
    """Steps of single tokens, of parts and their join, of prompts, and of both kinds in one
    launch (which asks for more LDS, on each device), while another device is current."""
    got = on_stub("""
steps = [([20, 5], [1, 1]), ([16000], [1]), ([700], [700]), ([700, 20], [700, 1])]
got = []
for on in (2, 3):
    stub.hipSetDevice(on)
    plans = [plan(*s) for s in steps]
    units = stub.stub_units_asked_of()
    stub.hipSetDevice(0)
    rcs = [attend(p) for p in plans]
    got.append([rcs, units, device(), stub.stub_lds_asked_on(), launches()])
    stub.stub_forget()
stub.stub_devices(3)
late = attend(plans[0])
print(json.dumps([got, late, stub.stub_launches(), ops.iekv_ops_last_error().decode()]))
""")
    for on, (rcs, units, current, lds, launches) in zip((2, 3), got[0]):
        assert rcs == [0, 0, 0, 0] and units == on and current == 0 and lds == 1 << on
        assert len(launches) >= 5 and {x[0] for x in launches} == {on}
        assert {x[4] for x in launches} == {77}
    # A device that is gone: an error, and nothing on another.
    assert got[1] == -2 and got[2] == 0 and "invalid device" in got[3]


class Elsewhere:
    """As much of a tensor on the second device as token_logprobs looks at."""

    is_cuda, requires_grad, device = True, False, torch.device("cuda", 1)

    def __init__(self, shape, dtype):
        self.shape, self.dtype = torch.Size(shape), dtype

    def dim(self):
        return len(self.shape)

    def stride(self, i):
        return (self.shape[-1], 1)[i]

    def is_neg(self):
        return False

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 4096

    def new_empty(self, shape, dtype):
        return torch.empty(shape, dtype=dtype)


def test_logprobs_run_on_the_logits_device(monkeypatch):
    from iekv.engine import logprobs

    current, ran_on = [0], []

    class Device:
        def __init__(self, device):
            self.index = torch.device(device).index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    monkeypatch.setattr(logprobs, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(logprobs, "current_stream_handle", lambda device: 0)
    monkeypatch.setattr(logprobs._ops, "entry",
                        lambda name: lambda *args: ran_on.append((name, current[0])) or 0)
    scored = logprobs.token_logprobs(Elsewhere((2, 100), torch.float32),
                                     Elsewhere((2,), torch.int64), top=3)
    assert scored.top_ids.shape == (2, 3)
    assert ran_on == [("iekv_logprobs", 1)] and current == [0]


def test_inputs_with_derivatives_are_refused():
    from torch.autograd import forward_ad

    from iekv.engine.pools import refuse_derivatives

    x = torch.ones(3)
    refuse_derivatives(x, "attend")
    with pytest.raises(RuntimeError, match="attend has no backward"):
        refuse_derivatives(x.clone().requires_grad_(), "attend")
    with torch.no_grad():
        refuse_derivatives(x.clone().requires_grad_(), "attend")
    with forward_ad.dual_level():
        refuse_derivatives(x, "attend")
        dual = forward_ad.make_dual(x, torch.ones(3))
        with pytest.raises(RuntimeError, match="forward mode"):
            refuse_derivatives(dual, "attend")
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward mode"):
            refuse_derivatives(dual * 2, "attend")
        refuse_derivatives(forward_ad.unpack_dual(dual).primal, "attend")


MOST = (2 ** 32 - 1) // 256          # workgroups of a launch


@pytest.mark.parametrize("rows, vocab, top, joins", [
    (MOST + 1, 5, 2, False), (2 * MOST + 3, 2000, 0, False), (MOST // 16 + 1, 128000, 3, True),
    (MOST // 2, 10000, 0, True), (MOST, 100, 1, False)])
def test_logprobs_of_many_rows_run_in_several_launches(on_stub, rows, vocab, top, joins):
    got = on_stub(f"""
A = 1 << 48
need = ops.iekv_logprobs_workspace(1, {rows}, {vocab}, {top})
rc = ops.iekv_logprobs(1, A, {vocab}, {rows}, {vocab}, 2 * A, {top}, 3 * A, 4 * A, 5 * A, 6 * A,
                       7 * A, need, 77)
print(json.dumps([rc, ops.iekv_ops_last_error().decode() if rc else "", launches()]))
""")
    rc, message, launches = got
    assert rc == 0, message
    parts, each = launches[::2 if joins else 1], 1 if not joins else -(-vocab // 8192)
    assert all(x[0] == 0 and x[4] == 77 and x[1] <= MOST for x in launches)
    assert sum(x[1] for x in parts) == rows * each
    if joins:
        assert len(launches) == 2 * len(parts)
        assert [-(-x[1] // each // 4) for x in parts] == [x[1] for x in launches[1::2]]


@pytest.mark.parametrize("step, blocks", [
    ("[1] * 16385, [1] * 16385", [16385 * 1024]),               # four heads a workgroup
    ("[17] * 4100, [17] * 4100", [4100 * 4096]),
    ("[17] * 4097 + [5], [17] * 4097 + [1]", [4097 * 4096, 4096]),   # not in one launch
    # Rows that are joined, four a workgroup: prompts of 120 behind a prefix worth sharing.
    ("[8312] * 140, [120] * 140, 16, 512", [None, 140 * 120 * 1024]),
])
def test_steps_of_any_size_run_in_several_launches(on_stub, step, blocks):
    got = on_stub(f"""
p = plan({step}, num_heads=4096, num_kv_heads=4096, head_dim=8)
rc = ops.iekv_attend(p, 1 << 44, 1 << 45, 1 << 46, 1 << 47, 4096 * 8, 8, 1.0, 3 << 46, 5 << 46,
                     1 << 46, 77)
print(json.dumps([rc, ops.iekv_ops_last_error().decode() if rc else "", launches()]))
""")
    rc, message, launches = got
    assert rc == 0, message
    assert all(x[0] == 0 and x[4] == 77 and x[1] <= MOST and x[2] == 1 for x in launches)
    total = sum(b for b in blocks if b is not None)
    if blocks[0] is None:
        assert sum(x[1] for x in launches) > total and launches[-1][1] == total - MOST
    else:
        assert sum(x[1] for x in launches) == total
    assert len(launches) > len(blocks) or blocks[-1] == 4096


def test_tables_that_are_missing_are_refused(on_stub):
    """Also where their lengths end at zero: a table is read by what it is said to hold."""
    got = on_stub("""
got = []
for starts, contexts in (([0, 2, 2], [20, 0]), ([0, 2, 0], [20, 0]), ([0, 0, 1], [0, 5])):
    out = ctypes.c_void_p()
    shape = _ops.AttentionShape(8, 2, 64, 16, 10, 3, 3, 0, 0, 0)
    rc = ops.iekv_attention_plan_create(
        ctypes.byref(shape), 2, (ctypes.c_int32 * 2)(*contexts), (ctypes.c_int32 * 2)(0, 0), None,
        (ctypes.c_int64 * 3)(*starts), ctypes.byref(out))
    got.append([rc, out.value, ops.iekv_ops_last_error().decode()])
out = ctypes.c_void_p()
rc = ops.iekv_attention_plan_create(
    ctypes.byref(shape), 2, (ctypes.c_int32 * 2)(0, 0), (ctypes.c_int32 * 2)(0, 0), None,
    (ctypes.c_int64 * 3)(0, 0, 0), ctypes.byref(out))
print(json.dumps([got, rc]))
""")
    for rc, plan, message in got[0]:
        assert rc == INVALID and plan is None and "tables is null" in message
    assert got[1] == 0
