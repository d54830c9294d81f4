"""KV pools in microscaled formats: quantised as they are written, read back as values.

The reference's caches hold the model's type (ie/kernels/reference.py:39-42,
ie/model/torch_transformer.py:82-86). A :class:`QuantizedPool` holds half of a 16-bit cache's
bytes, or a quarter: 32 dimensions of a head share a power of two, and an element is what is
left in 8 or 4 bits, rounded to nearest even.

    ``mxfp8``    e4m3: 3 bits after the leading one, off by 2^-4 of a value or, of small ones
                 beside a large one, by 2^-17 of the group's largest at most
    ``mxint8``   integers up to 127: off by 1/127 of the group's largest at most
    ``mxfp4``    e2m1: 1 bit after the leading one, off by 2^-2 of a value, or a twelfth of the
                 group's largest

The power is 2^-100 at least. Of a group too small for it elements are off by half a step there,
whatever they are of the largest: by 2^-110, 2^-101 and 2^-102. At the other end an element is
rounded past what a type of 16 or 32 bits holds, where reading it back in that type gives an
infinity, as its own rounding does: in float16 from 63,488 on (``mxfp8``), past 65,024
(``mxint8``) and from 57,344 on (``mxfp4``), though a float16 row goes up to 65,504; in bfloat16
and float32 2^112 times that.

A head's record is its elements and four bytes of exponents, so that a cache is an ordinary
array ``[num_blocks * block_size, num_kv_heads, record]`` of bytes: the handoff, the offload
tier and the wire move its blocks as they move any other's.

    k, v = allocate_quantized_pool(num_blocks, 16, layers, kv_heads, head_dim, format="mxfp8")
    pool = QuantizedPool(k, v, 16, "mxfp8")
    write_slots(pool, layer, k_rows, v_rows, slots)          # iekv.engine.slots
    plan = AttentionPlan(pool, tables, contexts, queries, num_heads)
    out = attend(plan, layer, q)                             # iekv.engine.attention
    rows = gather_rows(pool, layer, table, context_len, dtype=torch.bfloat16)

Records of two formats may be of the same size, so what moves them carries the format: copiers
(``HipSlotCopier(..., format=...)``, or an engine's of a model with a ``cache_format``), their
payloads and the wire's header. Blocks go only where the format is the same.
"""
from __future__ import annotations

import ctypes
import operator
from array import array as _ints
from typing import Sequence as Seq

import numpy as np
import torch

from .. import _native, _ops
from .pools import (KVPool, allocate_pool, allocate_pool_pair, current_device,
                    current_stream_handle, integer_ids, refuse_derivatives)

FORMATS = {"mxfp8": _ops.IEKV_TYPE_MXFP8, "mxint8": _ops.IEKV_TYPE_MXINT8,
           "mxfp4": _ops.IEKV_TYPE_MXFP4}
_CODE_BITS = {"mxfp8": 8, "mxint8": 8, "mxfp4": 4}
_SCALE_BYTES = 4

# Longest host lists of slots and host block tables that the library carries in its launches'
# arguments, in two launches; longer ones are uploaded.
HOST_SLOTS_MAX = 2 * _ops.MX_INLINE_SLOTS
HOST_TABLE_MAX = 2 * _ops.MX_INLINE_BLOCKS

_TYPES = {torch.float32: _native.IEKV_TYPE_F32, torch.float16: _native.IEKV_TYPE_F16,
          torch.bfloat16: _native.IEKV_TYPE_BF16}


def _known(format: str) -> None:
    if format not in FORMATS:
        raise ValueError(f"no format {format!r}: one of {', '.join(FORMATS)}")


def record_bytes(format: str, head_dim: int) -> int:
    """Bytes of one head of one token: its elements and the groups' exponents."""
    _known(format)
    if not 8 <= head_dim <= _ops.ATTENTION_MAX_DIM or head_dim % 8:
        raise ValueError(f"head_dim {head_dim} is not a multiple of 8 up to "
                         f"{_ops.ATTENTION_MAX_DIM}")
    return head_dim * _CODE_BITS[format] // 8 + _SCALE_BYTES


def head_dim_of(pool: KVPool, format: str) -> int:
    """The head dimension of the records that ``pool``'s caches hold; ValueError where they
    can hold none of ``format``."""
    _known(format)
    if pool.dtype != torch.uint8 or len(pool.tile_shape) != 3:
        raise ValueError(f"caches of records are [rows, KV heads, record] uint8, got tiles of "
                         f"{pool.tile_shape} {pool.dtype}")
    record = pool.tile_shape[2]
    head_dim = (record - _SCALE_BYTES) * 8 // _CODE_BITS[format]
    try:
        fits = record_bytes(format, head_dim) == record
    except ValueError:
        fits = False
    if not fits:
        raise ValueError(f"records of {record} bytes are none of {format}: head_dim is a "
                         f"multiple of 8 up to {_ops.ATTENTION_MAX_DIM}")
    return head_dim


def allocate_quantized_pool(num_blocks: int, block_size: int, num_layers: int,
                            num_kv_heads: int, head_dim: int, *, format: str,
                            device: str | torch.device = "cuda", zero: bool = True
                            ) -> tuple[list[torch.Tensor], list[torch.Tensor]]:
    """Per-layer K and V caches of records, views of one slab (zero-filled: every value 0)."""
    return allocate_pool(num_blocks, block_size, num_layers, num_kv_heads,
                         record_bytes(format, head_dim), dtype=torch.uint8, device=device,
                         zero=zero)


def allocate_quantized_pool_pair(first_blocks: int, second_blocks: int, block_size: int,
                                 num_layers: int, num_kv_heads: int, head_dim: int, *,
                                 format: str, device: str | torch.device = "cuda",
                                 zero: bool = True):
    """Two such pools in one allocation (:func:`iekv.engine.pools.allocate_pool_pair`)."""
    return allocate_pool_pair(first_blocks, second_blocks, block_size, num_layers, num_kv_heads,
                              record_bytes(format, head_dim), dtype=torch.uint8, device=device,
                              zero=zero)


class QuantizedPool(KVPool):
    """A registered set of per-layer caches whose rows are records of ``format``.

    ``k_caches`` and ``v_caches`` are ``[rows, num_kv_heads, record]`` uint8, as
    :func:`allocate_quantized_pool` makes them. The slot calls of :mod:`iekv.engine.slots` and
    the attention of :mod:`iekv.engine.attention` take and return values; the copiers move the
    records.
    """

    def __init__(self, k_caches: Seq[torch.Tensor], v_caches: Seq[torch.Tensor],
                 block_size: int, format: str) -> None:
        _known(format)
        super().__init__(k_caches, v_caches, block_size)
        head_dim, heads = head_dim_of(self, format), self.tile_shape[1]
        self.format = format
        self.num_kv_heads = heads
        self.head_dim = head_dim
        # What each call hands the library.
        self._shape = _ops.MxCache(FORMATS[format], heads, head_dim, block_size, self.num_blocks)
        self._shape_ref = ctypes.byref(self._shape)
        self._addresses = (ctypes.c_uint64 * len(self._ptrs))(*self._ptrs)
        self._at = ctypes.addressof(self._addresses)       # K of each layer, then V
        self._index = self._arrays[0].get_device()
        self._write = _ops.entry("iekv_mx_write_slots")
        self._write_ids = _ops.entry("iekv_mx_write_slots_ids")
        self._read = _ops.entry("iekv_mx_read_rows")
        self._read_ids = _ops.entry("iekv_mx_read_rows_ids")

    def _rows(self, t: torch.Tensor, what: str) -> torch.Tensor:
        """Rows as the library reads them: as they are where their heads are contiguous."""
        if t.get_device() != self._index:
            raise ValueError(f"{what} on {t.device}, pool on {self.device}")
        if t.dtype not in _TYPES:
            raise ValueError(f"{what} of {t.dtype}: float32, float16 or bfloat16 are quantised")
        refuse_derivatives(t, "a quantised cache")
        if t.is_neg():
            t = t.resolve_neg()
        return t if t.stride(-1) == 1 else t.contiguous()

    def _slots(self, slots, n: int):
        """The slots of n rows and the entry point that takes them: a device tensor as it is,
        host ones checked, and long lists uploaded."""
        if isinstance(slots, torch.Tensor) and slots.get_device() >= 0:
            if slots.get_device() != self._index:
                raise ValueError(f"slots on {slots.device}, pool on {self.device}")
            if slots.dtype != torch.int64:
                if slots.dtype.is_floating_point or slots.dtype.is_complex or \
                        slots.dtype == torch.bool:
                    raise TypeError(f"slots must be integers, not {slots.dtype}")
                slots = slots.to(torch.int64)
            if slots.dim() != 1 or slots.shape[0] != n:
                raise ValueError(f"slots of shape {tuple(slots.shape)} for {n} rows")
            return slots if slots.is_contiguous() else slots.contiguous(), self._write
        host = integer_ids(slots, "slot")
        if host.size != n:
            raise ValueError(f"{host.size} slots for {n} rows")
        rows = self.num_blocks * self.block_size
        bad = host[(host < 0) | (host >= rows)]
        if bad.size:
            raise IndexError(f"slot {bad[0]} out of range for a pool of {rows} slots")
        if np.unique(host).size != host.size:
            raise ValueError("slots must be distinct")
        if n <= HOST_SLOTS_MAX:
            return np.ascontiguousarray(host), self._write_ids
        return self._upload(host, f"a list of {n} slots"), self._write

    def _table(self, block_table, context_len: int):
        """The entries of a block table that a context uses, and the entry point that takes
        them."""
        if context_len < 0:
            raise ValueError(f"context of {context_len} rows")
        needed = -(-context_len // self.block_size)
        on_device = isinstance(block_table, torch.Tensor) and block_table.get_device() >= 0
        held = block_table.shape[0] if on_device else len(block_table)
        if held < needed:
            raise IndexError(f"context of {context_len} needs {needed} blocks, table has {held}")
        if on_device:
            if block_table.get_device() != self._index:
                raise ValueError(f"block table on {block_table.device}, pool on {self.device}")
            if block_table.dim() != 1 or block_table.dtype not in (torch.int32, torch.int64):
                raise TypeError(f"a device block table must be int32 or int64 in one dimension, "
                                f"got {tuple(block_table.shape)} {block_table.dtype}")
            if block_table.dtype == torch.int32 and block_table.is_contiguous():
                return block_table, self._read         # entries past the context are not read
            if block_table.dtype == torch.int64:       # outside the pool in 32 bits too
                block_table = block_table.clamp(-1, self.num_blocks)
            return block_table[:needed].to(torch.int32).contiguous(), self._read
        host = self.host_ids(block_table[:needed], what="context block")
        if host.size != needed:
            raise ValueError(f"a block table of {host.size} entries for {needed} blocks")
        host = host.astype(np.int32)
        if needed <= HOST_TABLE_MAX:
            return host, self._read_ids
        return self._upload(host, f"a table of {needed} blocks"), self._read

    def _upload(self, host: np.ndarray, what: str) -> torch.Tensor:
        with torch.cuda.device(self.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"{what} is uploaded, which a stream under capture cannot do: "
                                   "pass a device tensor")
            return torch.from_numpy(np.ascontiguousarray(host)).pin_memory().to(
                self.device, non_blocking=True)

    def _call(self, f, *args) -> None:
        """Call an entry point with the pool's shape first and its stream last, on its device."""
        stream = current_stream_handle(self.device)
        if self._index == current_device():
            code = f(self._shape_ref, *args, stream)
        else:
            with torch.cuda.device(self.device):
                code = f(self._shape_ref, *args, stream)
        if code:
            _ops.fail(f.__name__, code)


def _address(ids) -> int:
    return ids.data_ptr() if isinstance(ids, torch.Tensor) else ids.ctypes.data


def write(pool: QuantizedPool, first_layer: int, k: torch.Tensor, v: torch.Tensor,
          slots) -> None:
    """``[n_layers, n, H, D]`` rows into the slots of layers ``first_layer`` and on."""
    n_layers, n, heads, dim = k.shape
    if heads != pool.num_kv_heads or dim != pool.head_dim:
        raise ValueError(f"rows of shape {(heads, dim)} do not fit a pool of "
                         f"{(pool.num_kv_heads, pool.head_dim)}")
    k, v = pool._rows(k, "K rows"), pool._rows(v, "V rows")
    if k.dtype != v.dtype:
        raise ValueError(f"K rows of {k.dtype} and V rows of {v.dtype}")
    where, entry = pool._slots(slots, n)
    first_layer = operator.index(first_layer)      # NumPy's too: an address is made of it
    if first_layer < 0 or first_layer + n_layers > pool.num_layers:
        raise IndexError(f"layers {first_layer}..{first_layer + n_layers - 1} out of range for "
                         f"{pool.num_layers} layers")
    strides = _ints("q", (*k.stride(), *v.stride()))
    at = strides.buffer_info()[0]
    arrays = pool._at + 8 * first_layer            # K's; V's follow them
    pool._call(entry, arrays, arrays + 8 * pool.num_layers, n_layers, _TYPES[k.dtype],
               k.data_ptr(), at, v.data_ptr(), at + 32, _address(where), n)


def read(pool: QuantizedPool, first_array: int, n_arrays: int, block_table, context_len: int,
         dtype: torch.dtype | None) -> torch.Tensor:
    """``[n_arrays, context_len, H, D]`` values of a context (default: bfloat16)."""
    kind = _TYPES.get(torch.bfloat16 if dtype is None else dtype)
    if kind is None:
        raise ValueError(f"values of {dtype}: float32, float16 or bfloat16 are read back")
    context_len = operator.index(context_len)
    first_array, n_arrays = operator.index(first_array), operator.index(n_arrays)
    if first_array < 0 or n_arrays <= 0 or first_array + n_arrays > pool.n_arrays:
        raise IndexError(f"arrays {first_array}..{first_array + n_arrays - 1} out of range for "
                         f"{pool.n_arrays} arrays")
    table, entry = pool._table(block_table, context_len)
    out = torch.empty((n_arrays, context_len, pool.num_kv_heads, pool.head_dim),
                      dtype=torch.bfloat16 if dtype is None else dtype, device=pool.device)
    pool._call(entry, pool._at + 8 * first_array, n_arrays, _address(table), context_len, kind,
               out.data_ptr())
    return out
