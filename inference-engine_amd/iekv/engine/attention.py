"""Attention over the paged KV cache, through libiekv_ops.

An :class:`AttentionPlan` holds what the layers of a step have in common: the sequences'
block tables on the device and how their rows and keys are cut into workgroups.
:func:`attend` is one layer's attention by that plan. Queries are the last tokens of each
sequence's context, as the paged attention of the reference's step has it
(ie/kernels/reference.py:54-63 gathers the same rows first): a single token in a decode
step, a prompt or a chunk of one in a prefill step.

    plan = AttentionPlan(pool, layout.block_tables, layout.context_lens, layout.query_lens,
                         num_heads, window=4096, sinks=4)
    for layer in range(pool.num_layers):
        out = attend(plan, layer, q)              # q, out: [tokens, num_heads, head_dim]

A query at position ``p`` sees the keys ``j <= p`` with ``j > p - window`` or
``j < sinks``; without a window every key up to its own. ``shared_blocks`` says that every
block table begins with the same so many blocks, as the block manager's prefix sharing
makes them: where that saves more than it costs, their keys are read and scored once for all
sequences' queries together. The result is the same, up to rounding.

Forward only: the package serves and trains nothing, and queries that require a gradient or
carry a tangent are refused.
"""
from __future__ import annotations

import ctypes
import math
from array import array as _ints

import torch

from .. import _native, _ops
from .pools import KVPool, current_stream_handle, integer_ids, refuse_derivatives

_TYPES = {torch.float32: _native.IEKV_TYPE_F32, torch.float16: _native.IEKV_TYPE_F16,
          torch.bfloat16: _native.IEKV_TYPE_BF16, torch.float8_e4m3fn: _native.IEKV_TYPE_E4M3}


def _lengths(values, what: str) -> _ints:
    try:
        return _ints("i", values if type(values) in (list, tuple) else
                     integer_ids(values, what).tolist())
    except OverflowError:
        raise ValueError(f"{what} out of range") from None


def _flat_tables(block_tables, context_lens: _ints, block_size: int):
    """The used entries of every table end to end, and where each one's begin."""
    flat, starts = _ints("i"), _ints("q", [0])
    for table, context in zip(block_tables, context_lens):
        if isinstance(table, torch.Tensor) and table.device.type != "cpu":
            raise TypeError("block tables are host lists, arrays or CPU tensors")
        used = table[:max(0, -(-context // block_size))]
        try:
            flat.extend(_ints("i", used) if type(used) in (list, tuple) else
                        _ints("i", integer_ids(used).tolist()))
        except TypeError:               # not integers: refused as elsewhere
            flat.extend(_ints("i", integer_ids(used).tolist()))
        except OverflowError:
            raise IndexError("block id out of range") from None
        starts.append(len(flat))
    return flat, starts


def common_blocks(block_tables, context_lens, block_size: int) -> int:
    """How many leading blocks, filled by every context, all the block tables share."""
    tables = [list(t[:n // block_size]) for t, n in zip(block_tables, context_lens)]
    if len(tables) < 2:
        return 0
    shared = 0
    for column in zip(*tables):
        if column.count(column[0]) != len(column):
            break
        shared += 1
    return shared


class AttentionPlan:
    """How one step's attention over ``pool`` is done, for every layer.

    ``block_tables`` (host lists or arrays; entries past a context are not read),
    ``context_lens`` and ``query_lens`` are the step's, per sequence; a sequence without
    queries takes no part. ``query_dtype`` is the queries' type: float32 on any cache,
    float16 or bfloat16 on a cache of the same type or float8_e4m3fn (default: the cache's
    type, bfloat16 on an fp8 cache). IndexError for a block outside the pool or a table
    too short for its context, ValueError for tables that do not begin with the shared
    blocks and for arguments out of range.

    Making one costs the host 20-45 us for a few sequences, 220 us for 48 of 6,000 tokens in
    blocks of 16 and 400 us for 128 of 4,200, most of it to flatten the tables.

    The plan is uploaded on the device's current stream when it is made; :func:`attend`
    on another stream waits for that. A plan used in a captured graph has to live as long as
    the graph, and has to be made before the capture.
    """

    def __init__(self, pool: KVPool, block_tables, context_lens, query_lens, num_heads: int, *,
                 window: int | None = None, sinks: int = 0, shared_blocks: int = 0,
                 query_dtype: torch.dtype | None = None) -> None:
        if len(pool.tile_shape) != 3:
            raise ValueError(f"attention needs caches of [rows, KV heads, head_dim], got tiles "
                             f"of {pool.tile_shape}")
        if window is not None and window < 1:
            raise ValueError(f"window {window} must be at least 1 (None for no window)")
        if query_dtype is None:
            query_dtype = torch.bfloat16 if pool.dtype == torch.float8_e4m3fn else pool.dtype
        if query_dtype not in _TYPES or pool.dtype not in _TYPES:
            raise ValueError(f"attention of {query_dtype} queries on a {pool.dtype} cache")
        if not len(block_tables) == len(context_lens) == len(query_lens):
            raise ValueError(f"{len(block_tables)} block tables for {len(context_lens)} contexts "
                             f"and {len(query_lens)} query lengths")
        contexts = _lengths(context_lens, "context lengths")
        queries = _lengths(query_lens, "query lengths")
        flat, starts = _flat_tables(block_tables, contexts, pool.block_size)
        _, kv_heads, dim = pool.tile_shape
        shape = _ops.AttentionShape(num_heads, kv_heads, dim, pool.block_size, pool.num_blocks,
                                    _TYPES[query_dtype], _TYPES[pool.dtype],
                                    min(window or 0, 1 << 40), min(sinks, 1 << 40),
                                    shared_blocks)
        with torch.cuda.device(pool.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("an attention plan is uploaded, which a stream under capture "
                                   "cannot do: make it before the capture")
            self._handle = ctypes.c_void_p()
            # For the device that is current: attend runs there.
            _ops.call("iekv_attention_plan_create", ctypes.byref(shape), len(contexts),
                      contexts.buffer_info()[0], queries.buffer_info()[0],
                      flat.buffer_info()[0], starts.buffer_info()[0],
                      ctypes.byref(self._handle))
        self.pool = pool
        self.num_heads = num_heads
        self.query_dtype = query_dtype
        self.head_dim = dim
        words, n = ctypes.POINTER(ctypes.c_int32)(), ctypes.c_int64()
        tokens, workspace = ctypes.c_int64(), ctypes.c_int64()
        _ops.call("iekv_attention_plan_info", self._handle, ctypes.byref(words), ctypes.byref(n),
                  ctypes.byref(tokens), ctypes.byref(workspace))
        self.num_tokens = tokens.value
        self._workspace_bytes = workspace.value
        self._words = None
        if n.value:
            host = torch.empty(n.value, dtype=torch.int32, pin_memory=True)
            ctypes.memmove(host.data_ptr(), words, 4 * n.value)
            self._words = host.to(pool.device, non_blocking=True)
        self._words_at = self._words.data_ptr() if n.value else None
        # What attend needs of these for each call.
        self._shape = torch.Size((self.num_tokens, num_heads, dim))
        self._scale = 1.0 / math.sqrt(dim)
        self._attend = _ops.entry("iekv_attend")
        self._stream = current_stream_handle(pool.device)
        self._uploaded = torch.cuda.Event()
        self._uploaded.record(torch.cuda.current_stream(pool.device))
        # What attend hands the library for each layer.
        arrays = pool._ptrs
        self._layers = list(zip(arrays[:pool.num_layers], arrays[pool.num_layers:]))

    def __del__(self) -> None:
        try:
            if self._handle.value and _ops._lib is not None:
                _ops._lib.iekv_attention_plan_destroy(self._handle)
            self._handle = ctypes.c_void_p()
        except Exception:
            pass

    def _used_on(self, stream: int) -> None:
        """Order a stream other than the plan's own after the upload, and keep the plan's
        device memory until that stream has used it. A stream under capture is not made to
        wait: the capture began after the upload, and the caller orders its replays."""
        current = torch.cuda.current_stream(self.pool.device)
        with torch.cuda.device(self.pool.device):
            if torch.cuda.is_current_stream_capturing():
                return
        current.wait_event(self._uploaded)
        if self._words is not None:
            self._words.record_stream(current)


def attend(plan: AttentionPlan, layer: int, q: torch.Tensor, *, scale: float | None = None,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """The attention of ``layer`` for the plan's queries.

    ``q``: ``[tokens, num_heads, head_dim]`` on the pool's device, the sequences' queries
    one after the other, head ``h`` reading KV head ``h // (num_heads / kv_heads)``; any
    strides (a last dimension that is not contiguous is copied first). ``scale`` defaults to
    ``1 / sqrt(head_dim)``. Returns ``out``, or a new contiguous tensor of q's shape and
    type; ``out`` may be ``q`` itself, and overlap it in no other way. Runs on the
    current stream of the pool's device, whichever device is current.
    """
    pool = plan.pool
    device, shape = pool.device, plan._shape
    if q.dtype != plan.query_dtype or q.device != device:
        raise ValueError(f"queries of {q.dtype} on {q.device}, the plan is for "
                         f"{plan.query_dtype} on {device}")
    if q.shape != shape:
        raise ValueError(f"queries of shape {tuple(q.shape)}, the plan is for {tuple(shape)}")
    if not 0 <= layer < pool.num_layers:
        raise IndexError(f"layer {layer} out of range for {pool.num_layers} layers")
    refuse_derivatives(q, "attend")
    if q.is_neg():
        q = q.resolve_neg()
    if q.is_contiguous():
        token_stride, head_stride = shape[1] * shape[2], shape[2]
    else:
        if q.stride(2) != 1:
            q = q.contiguous()
        token_stride, head_stride = q.stride(0), q.stride(1)
    if out is None:
        out = q.new_empty(shape)
    elif out.shape != shape or out.dtype != q.dtype or out.device != device or \
            not out.is_contiguous() or out.is_neg():
        raise ValueError("out must be a contiguous tensor of the queries' shape, type and device")
    if not shape[0]:
        return out
    stream = current_stream_handle(device)
    if stream != plan._stream:
        plan._used_on(stream)
    need, workspace = plan._workspace_bytes, None
    if need:
        workspace = q.new_empty(need, dtype=torch.uint8)
    k, v = plan._layers[layer]
    code = plan._attend(plan._handle, plan._words_at, k, v, q.data_ptr(), token_stride, head_stride,
                        plan._scale if scale is None else scale, out.data_ptr(),
                        workspace.data_ptr() if need else None, need, stream)
    if code:
        _ops.fail("iekv_attend", code)
    return out
