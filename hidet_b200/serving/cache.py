"""The quantized, paged key/value cache: int8 codes with one float32 scale per token and head, for keys and for values.

    cache = quantized_cache(pages=1024, kv_heads=8, head_dim=128)                      # zeroed: empty
    q = quantized_cache_append(cache, k, v, slots, q=q, positions=positions, table=table)   # rotates q and k, stores k and v
    k, v = quantized_cache_read(cache, slots)                                          # rows of it back

A slot is page * page_size + the place in the page.  The tensor is uint8 [pages, kv_heads, page_size / 16, 32 head_dim + 128]; pages are whole runs of
memory, so they can be copied, swapped out and shared as such.  Its records are laid out for the attention kernel's copies
(include/hidet_b200q.h has the layout); rows are written and read with the functions here.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import ffi, native
from ..runtime import FLOAT_CODES, current_stream_ptr, require_cuda
from .rotary import LAYOUTS, check_index, check_table, heads_of, heads_struct

HEAD_DIMS = (64, 96, 128, 192, 256)


def quantized_cache(pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device='cuda') -> torch.Tensor:
    """An empty cache.  Takes 2 head_dim + 8 bytes for a position of a head (of 4 head_dim in 16 bits)."""
    if head_dim not in HEAD_DIMS:
        raise ValueError('heads of {} elements: {} are supported'.format(head_dim, ', '.join(map(str, HEAD_DIMS))))
    if page_size <= 0 or page_size % 16 != 0 or page_size > 65536:
        raise ValueError('pages of {} positions: multiples of 16 up to 65536 are supported'.format(page_size))
    if pages < 0 or kv_heads <= 0:
        raise ValueError('a cache of {} pages and {} heads'.format(pages, kv_heads))
    return torch.zeros((pages, kv_heads, page_size // 16, 32 * head_dim + 128), dtype=torch.uint8, device=device)


def cache_shape(cache: torch.Tensor) -> Tuple[int, int, int, int]:
    """(pages, kv_heads, page_size, head_dim) of a cache, which it checks."""
    require_cuda(cache, 'cache')
    dim = (cache.shape[-1] - 128) // 32 if cache.dim() == 4 else 0
    if cache.dtype != torch.uint8 or dim not in HEAD_DIMS or cache.shape[-1] != 32 * dim + 128 or not cache.is_contiguous():
        raise ValueError('expect a contiguous cache made by quantized_cache, got {} {}'.format(cache.dtype, list(cache.shape)))
    return cache.shape[0], cache.shape[1], cache.shape[2] * 16, dim


def quantized_cache_append(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, q: Optional[torch.Tensor] = None,
                           positions: Optional[torch.Tensor] = None, table: Optional[torch.Tensor] = None, layout: str = 'half') -> Optional[torch.Tensor]:
    """Quantizes k and v [..., kv_heads, head_dim] (float16, bfloat16 or float32, any strides between heads) into slots [...] of the cache: per row,
    code = rint(x * (127 / amax)), scale = amax / 127.  Negative slots are passed over (padding); one beyond the cache is passed over and reported
    by b200q_check_status.  The slots of one call differ.

    With positions [...] and a table (rotary_table) k is rotated on the way, and q [..., heads, head_dim], if given, is rotated and returned: what
    rotary_embedding and an append do, in one launch, with k quantized before it is rounded to 16 bits."""
    rotated = native.append(cache, k, v, slots, q, positions, table, layout)
    if rotated is not None:
        return rotated if q is not None else None
    pages, kv_heads, page_size, dim = cache_shape(cache)
    require_cuda(k, 'k')
    require_cuda(v, 'v')
    if k.dtype not in FLOAT_CODES or v.dtype != k.dtype or k.device != cache.device or v.device != cache.device:
        raise ValueError('expect k and v of one type (float16, bfloat16 or float32) on {}, got {} on {} and {} on {}'.format(cache.device, k.dtype, k.device, v.dtype, v.device))
    if layout not in LAYOUTS:
        raise ValueError("layout must be 'half' or 'interleaved', got {!r}".format(layout))
    lead = list(k.shape[:-2])
    for x, name in ((k, 'k'), (v, 'v')):
        if x.dim() < 2 or list(x.shape) != lead + [kv_heads, dim]:
            raise ValueError('{} has shape {}, expected {}'.format(name, list(x.shape), lead + [kv_heads, dim]))
    slots = check_index(slots, 'slots', lead, cache.device)
    if (positions is None) != (table is None) or (q is not None and positions is None):
        raise ValueError('a rotation needs positions and a table')
    rotary_dim = table_rows = position_bytes = 0
    if table is not None:
        table = check_table(table, cache.device, dim)
        table_rows, rotary_dim = table.shape
        if rotary_dim % 16 != 0:
            raise ValueError('{} rotated elements: multiples of 16 are supported here (rotary_embedding takes others)'.format(rotary_dim))
        positions = check_index(positions, 'positions', lead, cache.device)
        position_bytes = positions.element_size()
    out = qs = outs = None
    if q is not None:
        require_cuda(q, 'q')
        if q.dtype != k.dtype or q.device != cache.device:
            raise ValueError('q is {} on {}, k {} on {}'.format(q.dtype, q.device, k.dtype, k.device))
        q2, heads = heads_of(q, 'q', lead, dim)
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        qs, outs = heads_struct(q2), heads_struct(heads_of(out, 'q', lead, dim)[0])
    k2, v2 = heads_of(k, 'k', lead, dim)[0], heads_of(v, 'v', lead, dim)[0]
    with torch.cuda.device(cache.device):
        ffi.func('b200q_quantized_cache_append')(
            cache.data_ptr(), pages, page_size, heads_struct(k2), heads_struct(v2), qs, outs, slots.data_ptr(), positions.data_ptr() if positions is not None else None,
            table.data_ptr() if table is not None else None, slots.numel(), q.shape[-2] if q is not None else 0, kv_heads, dim, rotary_dim, table_rows, LAYOUTS[layout],
            FLOAT_CODES[k.dtype], slots.element_size(), position_bytes, current_stream_ptr(cache.device))
    return out


def quantized_cache_read(cache: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [..., kv_heads, head_dim]: the rows in slots [...], code * scale rounded to dtype once.  Zeros for a negative slot and for one beyond the
    cache, which b200q_check_status reports."""
    pair = native.read(cache, slots, dtype)
    if pair is not None:
        return pair
    pages, kv_heads, page_size, dim = cache_shape(cache)
    if dtype not in FLOAT_CODES:
        raise ValueError('quantized_cache_read gives float16, bfloat16 or float32, not {}'.format(dtype))
    require_cuda(slots, 'slots')
    slots = check_index(slots, 'slots', slots.shape, cache.device)
    k, v = (torch.empty(list(slots.shape) + [kv_heads, dim], dtype=dtype, device=cache.device) for _ in 'kv')
    with torch.cuda.device(cache.device):
        ffi.func('b200q_quantized_cache_read')(cache.data_ptr(), pages, page_size, slots.data_ptr(), k.data_ptr(), v.data_ptr(), slots.numel(), kv_heads, dim,
                                               FLOAT_CODES[dtype], slots.element_size(), current_stream_ptr(cache.device))
    return k, v
