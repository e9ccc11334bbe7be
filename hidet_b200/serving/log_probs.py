"""Log probabilities of given tokens with the entropy and the top alternatives of every row, in one pass over the logits."""
from __future__ import annotations

from typing import Tuple

import torch

from .. import ffi, native
from ..runtime import FLOAT_CODES, current_stream_ptr, require_cuda
from .rotary import INDEX_TYPES

MOST_TOP = 32


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(log_probs, entropy, top_log_probs, top_indices) under softmax(logits[..., :]), all float32 but the int64 indices.

    logits [..., vocab] float16, bfloat16 or float32, rows of up to 1638400 bytes (409600 tokens in float32); tokens int32 or int64,
    [...] or [..., n] (n tokens of every row): log_probs has their shape.
    entropy [...] in nats; top_log_probs and top_indices [..., top] (top at most 32) the largest, descending, equal logits by index.
    -inf logits are tokens without probability; a row with a NaN or +inf, or of nothing but -inf, gives NaN.  A token outside the vocabulary has -inf and is
    reported by b200q_check_status."""
    result = native.log_probs(logits, tokens, top)
    if result is not None:
        return result
    require_cuda(logits, 'logits')
    require_cuda(tokens, 'tokens')
    if logits.dtype not in FLOAT_CODES or logits.dim() < 1:
        raise ValueError('token_log_probs expects float16, bfloat16 or float32 logits [..., vocab], got {} {}'.format(logits.dtype, list(logits.shape)))
    lead, vocab = list(logits.shape[:-1]), logits.shape[-1]
    if tokens.dtype not in INDEX_TYPES or list(tokens.shape[:len(lead)]) != lead or tokens.dim() > len(lead) + 1 or tokens.device != logits.device:
        raise ValueError('expect int32 or int64 tokens {0} or {0} + [n] on {1}, got {2} {3} on {4}'.format(lead, logits.device, tokens.dtype, list(tokens.shape), tokens.device))
    if not isinstance(top, int) or isinstance(top, bool) or not 0 <= top <= min(MOST_TOP, vocab):
        raise ValueError('top must be a whole number of 0 to {}, got {!r}'.format(min(MOST_TOP, vocab), top))
    given = tokens.shape[-1] if tokens.dim() > len(lead) else 1
    rows = logits.flatten(0, -2) if len(lead) > 1 else logits if lead else logits[None]
    if rows.stride(1) != 1 and vocab > 1:
        rows = rows.contiguous()
    if rows.shape[0] > 1 and rows.stride(0) < vocab:  # rows that overlap
        rows = rows.contiguous()
    tokens = tokens.contiguous()
    log_probs = torch.empty(tokens.shape, dtype=torch.float32, device=logits.device)
    entropy = torch.empty(lead, dtype=torch.float32, device=logits.device)
    values = torch.empty(lead + [top], dtype=torch.float32, device=logits.device)
    indices = torch.empty(lead + [top], dtype=torch.int64, device=logits.device)
    with torch.cuda.device(logits.device):
        ffi.func('b200q_token_log_probs')(rows.data_ptr(), rows.stride(0), tokens.data_ptr(), log_probs.data_ptr(), entropy.data_ptr(), values.data_ptr(), indices.data_ptr(),
                                          rows.shape[0], vocab, given, top, FLOAT_CODES[logits.dtype], tokens.element_size(), current_stream_ptr(logits.device))
    return log_probs, entropy, values, indices
