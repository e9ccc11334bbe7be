"""Attention of new tokens over the quantized cache: one token a sequence, several, or a tree of drafted ones."""
from __future__ import annotations

import math
from typing import Optional

import torch

from .. import ffi, native
from ..runtime import FLOAT_CODES, current_stream_ptr, require_cuda, workspaces
from .cache import cache_shape
from .rotary import heads_of, heads_struct


def quantized_cache_attention(q: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor] = None,
                              mask: Optional[torch.Tensor] = None, scale: Optional[float] = None, return_lse: bool = False):
    """softmax(scale * q k^T) v over the cached positions of every sequence, its newest tokens (the rows of q) among them.

    q           float16 or bfloat16: [batch, heads, dim], one token a sequence; [batch, t, heads, dim], t tokens each; or, with starts, [tokens, heads, dim],
                those of sequence b in rows starts[b] .. starts[b + 1] - 1 (int32 [batch + 1]).  heads is a multiple of the cache's.  Rows in front of
                starts[0] and from starts[batch] on, such as a captured step's unused ones, are zeros, with -inf for their denominators.
    page_table  int32 [batch, n]: the pages of every sequence, in order; lengths int32 [batch]: its cached positions, new tokens included.
    mask        None: a token sees every position up to its own.  Or bool / uint8 [tokens, w] with a row for every row of q: of the positions in front of its
                sequence's new tokens it sees all, and the j-th of these where mask[row, j] (w at least the most of a sequence).  Trees of drafted
                tokens are such masks.  A row that sees nothing is zeros.
    scale       a positive number, 1 / sqrt(dim) by default.
    Returns the result in q's shape and type, and with return_lse also the natural logarithm of the softmax's denominators, float32 of q's shape without dim.

    Everything that changes from step to step is on the device: a captured step can be replayed while the sequences grow.  Lengths beyond the page
    table are cut, and they and pages outside the cache are reported by b200q_check_status.  So are starts that fall or lie outside the rows; all rows are
    zeros then."""
    result = native.attention(q, cache, page_table, lengths, starts, mask, scale, return_lse)
    if result is not None:
        return result
    require_cuda(q, 'q')
    pages, kv_heads, page_size, dim = cache_shape(cache)
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError('quantized_cache_attention expects float16 or bfloat16 queries, got {}'.format(q.dtype))
    if q.dim() not in (3, 4) or (q.dim() == 4 and starts is not None) or q.shape[-1] != dim or q.shape[-2] == 0 or q.shape[-2] % kv_heads != 0:
        raise ValueError('q has shape {} (starts {}given), expected [batch, heads, {d}], [batch, t, heads, {d}] or, with starts, [tokens, heads, {d}], heads a multiple of {}'.format(
            list(q.shape), '' if starts is not None else 'not ', kv_heads, d=dim))
    heads = q.shape[-2]
    tensors = [('cache', cache), ('page_table', page_table), ('lengths', lengths)] + [(n, t) for n, t in (('starts', starts), ('mask', mask)) if t is not None]
    for name, t in tensors:
        require_cuda(t, name)
        if t.device != q.device:
            raise ValueError('{} is on {}, q on {}'.format(name, t.device, q.device))
    if lengths.dtype != torch.int32 or lengths.dim() != 1:
        raise ValueError('expect int32 lengths [batch], got {} {}'.format(lengths.dtype, list(lengths.shape)))
    batch = lengths.shape[0]
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != batch:
        raise ValueError('expect an int32 page table [{}, n], got {} {}'.format(batch, page_table.dtype, list(page_table.shape)))
    if starts is not None:
        if starts.dtype != torch.int32 or list(starts.shape) != [batch + 1]:
            raise ValueError('expect int32 starts [{}], got {} {}'.format(batch + 1, starts.dtype, list(starts.shape)))
        starts = starts.contiguous()
    elif q.shape[0] != batch:
        raise ValueError('{} sequences have lengths, {} have rows of q'.format(batch, q.shape[0]))
    rows, _ = heads_of(q, 'q', list(q.shape[:-2]), dim)
    if rows.data_ptr() % 16 != 0 or rows.stride(0) % 8 != 0 or rows.stride(1) % 8 != 0:
        rows = rows.clone(memory_format=torch.contiguous_format)  # loads of eight elements
    tokens = rows.shape[0]
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8) or mask.dim() != 2 or mask.shape[0] != tokens:
            raise ValueError('expect a bool or uint8 mask [{}, w], got {} {}'.format(tokens, mask.dtype, list(mask.shape)))
        if starts is None and mask.shape[1] < tokens // max(1, batch):
            raise ValueError('a mask of {} columns for {} tokens a sequence'.format(mask.shape[1], tokens // max(1, batch)))
        if mask.stride(1) != 1 and mask.shape[1] > 1:
            mask = mask.contiguous()
    if page_table.stride(1) != 1 and page_table.shape[1] > 1:
        page_table = page_table.contiguous()
    lengths = lengths.contiguous()
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device) if return_lse else None
    with torch.cuda.device(q.device):
        ws_ptr, ws_size = workspaces.get(q.device, ffi.func('b200q_quantized_cache_attention_workspace_bytes')(batch, tokens, heads, kv_heads, dim))
        ffi.func('b200q_quantized_cache_attention')(
            heads_struct(rows), out.data_ptr(), lse.data_ptr() if return_lse else None, cache.data_ptr(), pages, page_size, page_table.data_ptr(), page_table.shape[1],
            page_table.stride(0), lengths.data_ptr(), starts.data_ptr() if starts is not None else None, mask.data_ptr() if mask is not None else None,
            mask.shape[1] if mask is not None else 0, mask.stride(0) if mask is not None else 0, batch, tokens, heads, kv_heads, dim, scale, FLOAT_CODES[q.dtype],
            ws_ptr, ws_size, current_stream_ptr(q.device))
    return (out, lse) if return_lse else out
