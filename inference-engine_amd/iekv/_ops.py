"""ctypes binding of libiekv_ops.so: attention over the paged cache and the scoring of
answers (C-ABI in include/iekv_ops.h).

Loaded like the handoff library (:mod:`iekv._native`): after torch, with no fallback, and
with the same kinds of exception for the same status codes.
"""
from __future__ import annotations

import ctypes
import os
from ctypes import POINTER, c_char_p, c_float, c_int, c_int32, c_int64, c_void_p
from pathlib import Path

from . import _native

LIBRARY = Path(__file__).resolve().parent / "libiekv_ops.so"
ABI_VERSION = 1

ATTENTION_MAX_DIM = 128              # IEKV_ATTENTION_MAX_DIM
ATTENTION_MAX_GROUP = 128            # IEKV_ATTENTION_MAX_GROUP
ATTENTION_MAX_CONTEXT = 1 << 30      # IEKV_ATTENTION_MAX_CONTEXT
LOGPROBS_MAX_TOP = 64                # IEKV_LOGPROBS_MAX_TOP


class AttentionShape(ctypes.Structure):
    """iekv_attention_shape."""

    _fields_ = [("num_heads", c_int32), ("num_kv_heads", c_int32), ("head_dim", c_int32),
                ("block_size", c_int32), ("num_blocks", c_int64), ("query_type", c_int32),
                ("cache_type", c_int32), ("window", c_int64), ("sinks", c_int64),
                ("shared_blocks", c_int64)]


# Every entry point of include/iekv_ops.h: name -> (restype, argtypes).
SIGNATURES: dict[str, tuple[object, list[object]]] = {
    "iekv_ops_abi_version": (c_int, []),
    "iekv_ops_last_error": (c_char_p, []),
    "iekv_attention_plan_create": (c_int, [POINTER(AttentionShape), c_int32, c_void_p, c_void_p,
                                           c_void_p, c_void_p, POINTER(c_void_p)]),
    "iekv_attention_plan_destroy": (c_int, [c_void_p]),
    "iekv_attention_plan_info": (c_int, [c_void_p, POINTER(POINTER(c_int32)), POINTER(c_int64),
                                         POINTER(c_int64), POINTER(c_int64)]),
    "iekv_attend": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int64,
                            c_float, c_void_p, c_void_p, c_int64, c_void_p]),
    "iekv_logprobs_workspace": (c_int64, [c_int32, c_int64, c_int64, c_int32]),
    "iekv_logprobs": (c_int, [c_int32, c_void_p, c_int64, c_int64, c_int64, c_void_p, c_int32,
                              c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64,
                              c_void_p]),
}

_lib: ctypes.CDLL | None = None


def library_path() -> Path:
    override = os.environ.get("IEKV_OPS_LIBRARY")
    return Path(override) if override else LIBRARY


def lib() -> ctypes.CDLL:
    """The loaded library (loaded on first use)."""
    global _lib
    if _lib is not None:
        return _lib
    import torch  # noqa: F401  (binds the library to torch's HIP runtime)

    path = library_path()
    if not path.exists():
        raise RuntimeError(
            f"{path} is missing: build it with `python -m iekv.build` or "
            "`python -c 'import __graft_entry__ as g; g.build()'` before using the operators")
    handle = ctypes.CDLL(str(path))
    handle.iekv_ops_abi_version.restype, handle.iekv_ops_abi_version.argtypes = \
        SIGNATURES["iekv_ops_abi_version"]
    version = handle.iekv_ops_abi_version()
    if version != ABI_VERSION:
        raise RuntimeError(f"{path} has ABI version {version}, expected {ABI_VERSION}")
    for name, (restype, argtypes) in SIGNATURES.items():
        fn = getattr(handle, name)
        fn.restype = restype
        fn.argtypes = argtypes
    _lib = handle
    return handle


_functions: dict[str, ctypes._CFuncPtr] = {}


def entry(function: str) -> ctypes._CFuncPtr:
    """An entry point itself, for callers that are called often: pass a code other than 0
    to :func:`fail`."""
    f = _functions.get(function)
    if f is None:
        f = _functions[function] = getattr(lib(), function)
    return f


def fail(function: str, code: int) -> None:
    """Raise what :func:`iekv._native.call` raises for the code of a failed call."""
    message = lib().iekv_ops_last_error().decode(errors="replace")
    raise _native._ERRORS.get(code, _native.NativeError)(function, code, message)


def call(function: str, *args) -> None:
    """Call an entry point; raises as :func:`iekv._native.call` does."""
    code = entry(function)(*args)
    if code:
        fail(function, code)
