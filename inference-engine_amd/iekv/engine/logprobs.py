"""Log probabilities of given tokens, through libiekv_ops.

What an answer is scored with: for each row of logits the log probability of the token
that followed, the entropy of the distribution it was drawn from, and the most likely
alternatives. The reference draws its tokens from the logits on the host
(ie/layers/functional.py:64-73) and scores none.
"""
from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache

import torch

from .. import _native, _ops
from .pools import current_device, current_stream_handle, refuse_derivatives

_TYPES = {torch.float32: _native.IEKV_TYPE_F32, torch.float16: _native.IEKV_TYPE_F16,
          torch.bfloat16: _native.IEKV_TYPE_BF16}


@dataclass(slots=True)
class TokenLogprobs:
    """What :func:`token_logprobs` returns, on the logits' device."""

    logprobs: torch.Tensor        # [rows] float32: of the given token
    entropy: torch.Tensor         # [rows] float32, in nats
    top_logprobs: torch.Tensor    # [rows, top] float32, falling
    top_ids: torch.Tensor         # [rows, top] int64


@lru_cache(maxsize=256)
def _workspace_bytes(kind: int, rows: int, vocab: int, top: int) -> int:
    return _ops.lib().iekv_logprobs_workspace(kind, rows, vocab, top)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0) -> TokenLogprobs:
    """Score ``tokens[i]`` under ``softmax(logits[i])``, for every row.

    ``logits``: ``[rows, vocab]`` float32, float16 or bfloat16 on the GPU, any row stride;
    ``tokens``: ``[rows]`` int64 on the same device. ``top`` (at most 64) alternatives are
    ordered by logit, equal ones by index. Barred tokens (logits of -inf) have probability
    zero; a row that bars every token has log probabilities of -inf and entropy 0; a row with
    a NaN or +inf is NaN; a token outside the vocabulary (a padding mark) has log
    probability NaN. Runs on the current stream of the logits' device, whichever device is
    current.
    """
    if logits.dim() != 2 or logits.dtype not in _TYPES or not logits.is_cuda:
        raise ValueError(f"logits must be [rows, vocab] float32, float16 or bfloat16 on the GPU, "
                         f"got {tuple(logits.shape)} {logits.dtype} on {logits.device}")
    rows, vocab = logits.shape
    if tokens.shape != (rows,) or tokens.dtype != torch.int64 or tokens.device != logits.device:
        raise ValueError(f"tokens must be [{rows}] int64 on {logits.device}, got "
                         f"{tuple(tokens.shape)} {tokens.dtype} on {tokens.device}")
    if not 0 <= top <= min(vocab, _ops.LOGPROBS_MAX_TOP):
        raise ValueError(f"top {top} out of range for a vocabulary of {vocab} (at most "
                         f"{_ops.LOGPROBS_MAX_TOP})")
    if logits.device.index != current_device():
        with torch.cuda.device(logits.device):
            return token_logprobs(logits, tokens, top=top)
    refuse_derivatives(logits, "token_logprobs")
    if logits.stride(1) != 1 or logits.is_neg():
        logits = logits.contiguous().resolve_neg()
    if not tokens.is_contiguous() or tokens.is_neg():
        tokens = tokens.contiguous().resolve_neg()
    logprobs = logits.new_empty(rows, dtype=torch.float32)
    entropy = logits.new_empty(rows, dtype=torch.float32)
    top_logprobs = logits.new_empty((rows, top), dtype=torch.float32)
    top_ids = logits.new_empty((rows, top), dtype=torch.int64)
    if rows:
        kind = _TYPES[logits.dtype]
        need, workspace = _workspace_bytes(kind, rows, vocab, top), None
        if need:
            workspace = logits.new_empty(need, dtype=torch.uint8)
        code = _ops.entry("iekv_logprobs")(
            kind, logits.data_ptr(), logits.stride(0), rows, vocab, tokens.data_ptr(), top,
            logprobs.data_ptr(), entropy.data_ptr(), top_logprobs.data_ptr(), top_ids.data_ptr(),
            workspace.data_ptr() if need else None, need, current_stream_handle(logits.device))
        if code:
            _ops.fail("iekv_logprobs", code)
    return TokenLogprobs(logprobs, entropy, top_logprobs, top_ids)
