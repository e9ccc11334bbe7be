"""Rotary positions: the table of cosines and sines, made once, and the rotation of queries and keys.

    table = rotary_table(4096, 128)                                  # float32 [4096, 128]
    q, k = rotary_embedding(q, k, positions, table)                  # q [tokens, heads, 128], k [tokens, kv_heads, 128]
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from .. import ffi, native
from ..runtime import FLOAT_CODES, current_stream_ptr, require_cuda

LAYOUTS = {'half': ffi.ROTARY_HALF, 'interleaved': ffi.ROTARY_INTERLEAVED}
INDEX_TYPES = (torch.int32, torch.int64)


def rotary_table(positions: int, rotary_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                 original_positions: Optional[int] = None, device='cuda') -> torch.Tensor:
    """float32 [positions, rotary_dim]: of every position the cosines, then the sines, of position * base^(-2i / rotary_dim), computed in 64 bits.

    scaling lets a model made for original_positions (default: positions / factor) serve `factor` times as many:
        'linear'  positions divided by factor
        'ntk'     base * factor^(d / (d - 2)): the slowest pair turns factor times more slowly, the fastest as before
        'yarn'    pairs that make less than one turn in original_positions are slowed down by factor, those that make more than
                  32 stay, with a ramp between; cosines and sines times 0.1 ln(factor) + 1
    """
    if rotary_dim < 2 or rotary_dim % 2 != 0:
        raise ValueError('rotary_dim must be an even number from 2 on, got {}'.format(rotary_dim))
    if positions < 0:
        raise ValueError('positions must not be negative, got {}'.format(positions))
    if scaling not in (None, 'linear', 'ntk', 'yarn'):
        raise ValueError("scaling must be None, 'linear', 'ntk' or 'yarn', got {!r}".format(scaling))
    if not factor > 0 or not base > 1:
        raise ValueError('a positive factor and a base above 1 are wanted, got {} and {}'.format(factor, base))
    d, by = rotary_dim, 1.0
    if scaling == 'ntk':
        if d == 2:
            raise ValueError("scaling='ntk' needs more than one pair")
        base = base * factor ** (d / (d - 2))
    frequency = base ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    if scaling == 'linear':
        frequency = frequency / factor
    elif scaling == 'yarn':
        original = positions / factor if original_positions is None else original_positions

        def pair_of(turns):  # the pair (not a whole number) that makes so many turns in the original positions
            return d * math.log(max(original, 1) / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(pair_of(32.0)), 0), min(math.ceil(pair_of(1.0)), d - 1)
        ramp = ((torch.arange(d // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        frequency = frequency / factor * ramp + frequency * (1 - ramp)
        by = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * frequency.to(device)
    return torch.cat([angle.cos() * by, angle.sin() * by], -1).float()


def heads_of(t: torch.Tensor, name: str, lead, dim: Optional[int] = None) -> Tuple[torch.Tensor, int]:
    """(t as [tokens, heads, dim] with neighbouring elements, heads): `lead` are the dimensions of tokens."""
    if t.dim() != len(lead) + 2 or list(t.shape[:-2]) != list(lead) or (dim is not None and t.shape[-1] != dim):
        raise ValueError('{} has shape {}, expected {} + [heads, {}]'.format(name, list(t.shape), list(lead), 'dim' if dim is None else dim))
    if len(lead) != 1:
        t = t.flatten(0, len(lead) - 1) if lead else t[None]
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        t = t.contiguous()
    return t, t.shape[1]


def heads_struct(t: torch.Tensor) -> ffi.Heads:
    return ffi.Heads(t.data_ptr(), t.stride(0), t.stride(1))


def check_table(table: torch.Tensor, device, dim: int) -> torch.Tensor:
    require_cuda(table, 'table')
    if table.dtype != torch.float32 or table.dim() != 2 or table.shape[1] % 2 != 0 or not 2 <= table.shape[1] <= dim or table.device != device:
        raise ValueError('expect a float32 table [positions, rotary_dim] on {} with an even rotary_dim of at most {}, got {} {} on {}'.format(
            device, dim, table.dtype, list(table.shape), table.device))
    return table.contiguous()


def check_index(t: torch.Tensor, name: str, shape, device) -> torch.Tensor:
    require_cuda(t, name)
    if t.dtype not in INDEX_TYPES or list(t.shape) != list(shape) or t.device != device:
        raise ValueError('expect int32 or int64 {} of shape {} on {}, got {} {} on {}'.format(name, list(shape), device, t.dtype, list(t.shape), t.device))
    return t.contiguous()


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, table: torch.Tensor, layout: str = 'half',
                     out: Optional[Tuple[torch.Tensor, Optional[torch.Tensor]]] = None):
    """(q', k'): the first table.shape[1] elements of every head of q [..., heads, dim] and k [..., kv_heads, dim] (None: no keys) rotated by the
    angles of their token's position, the others copied.  q and k may be views into one projection's rows.

    layout says which elements are a pair: 'half' (i, i + rotary_dim / 2), 'interleaved' (2i, 2i + 1).  positions is int32 or int64 [...]; a position
    outside the table gives zeros and is reported by b200q_check_status.  `out` = (q', k') receives the result; out=(q, k) rotates in place.
    float32 arithmetic, one rounding to q's type (float16, bfloat16 or float32)."""
    if out is None:
        pair = native.rotary(q, k, positions, table, layout)
        if pair is not None:
            return pair
    require_cuda(q, 'q')
    if q.dtype not in FLOAT_CODES:
        raise ValueError('rotary_embedding expects float16, bfloat16 or float32, got {}'.format(q.dtype))
    if layout not in LAYOUTS:
        raise ValueError("layout must be 'half' or 'interleaved', got {!r}".format(layout))
    if q.dim() < 2:
        raise ValueError('q has shape {}, expected [..., heads, dim]'.format(list(q.shape)))
    lead, dim = list(q.shape[:-2]), q.shape[-1]
    table = check_table(table, q.device, dim)
    positions = check_index(positions, 'positions', lead, q.device)
    given = [q] if k is None else [q, k]
    if k is not None:
        require_cuda(k, 'k')
        if k.dtype != q.dtype or k.device != q.device:
            raise ValueError('k is {} on {}, q {} on {}'.format(k.dtype, k.device, q.dtype, q.device))
    sources = [heads_of(x, name, lead, dim)[0] for x, name in zip(given, 'qk')]
    if out is None:
        results = [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in given]
    else:
        results = [x for x in out if x is not None]
        if len(out) != 2 or len(results) != len(given) or any(
                y.shape != x.shape or y.dtype != x.dtype or y.device != x.device or (y.stride(-1) != 1 and dim > 1) for x, y in zip(given, results)):
            raise ValueError('out must be a pair of tensors like q and k with neighbouring elements')
        if any(stride == 0 and n > 1 for y in results for stride, n in zip(y.stride(), y.shape)):
            raise ValueError('out has elements that share their memory')
    targets = [heads_of(y, 'out', lead, dim)[0] for y in results]
    if any(t.untyped_storage().data_ptr() != y.untyped_storage().data_ptr() for t, y in zip(targets, results)):
        raise ValueError('the token dimensions of out cannot be viewed as one')
    structs = [heads_struct(t) for t in sources + targets]
    n = len(given)
    with torch.cuda.device(q.device):
        ffi.func('b200q_rotary_embedding')(
            structs[0], structs[1] if n == 2 else None, structs[n], structs[n + 1] if n == 2 else None, positions.data_ptr(), table.data_ptr(), positions.numel(),
            q.shape[-2], k.shape[-2] if k is not None else 0, dim, table.shape[1], table.shape[0], LAYOUTS[layout], FLOAT_CODES[q.dtype],
            positions.element_size(), current_stream_ptr(q.device))
    return results[0], results[1] if n == 2 else None
