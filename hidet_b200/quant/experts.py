"""A feed-forward layer of experts on int8 weights: decode steps and prompts.

    experts, weights = route_tokens(x, router, top_k=2)
    y = mixture_of_experts(x, experts, weights, gate_up, gate_up_scale, down, down_scale, residual=x)

The experts' weights are those of torch linears, side by side, quantized in one call over the last dimension:

    gate_up, gate_up_scale = symmetric_quantize(torch.stack((gate, up), 2).flatten(1, 2), 'int8', dims=-1)     # gate, up [experts, inner, hidden]
    down, down_scale = symmetric_quantize(down, 'int8', dims=-1)                                               # [experts, hidden, inner]

Not offered by the reference.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import ffi, native
from ..runtime import FLOAT_CODES, current_stream_ptr, require_cuda, workspaces
from .tokens import rows_of

MOST_EXPERTS, MOST_TOP = 1024, 32


def lines_of(rows: torch.Tensor) -> torch.Tensor:
    """Rows that begin on boundaries of 16 bytes, for loads of eight elements: a copy where they do not and a copy's would."""
    if rows.shape[1] % 8 != 0:
        return rows
    if rows.data_ptr() % 16 != 0 or (rows.stride(0) % 8 != 0 and rows.shape[0] > 1):
        return rows.clone(memory_format=torch.contiguous_format)
    return rows


def route_tokens(x: torch.Tensor, router: torch.Tensor, top_k: int, normalize: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """(experts, weights) [..., top_k], int32 and float32: the experts whose logits x @ router.T are the largest, descending, equal ones by index, and their shares of the
    softmax, over the chosen ones (normalize) or over all.

    x [..., hidden] float16, bfloat16 or float32; router [count, hidden] of x's type or float32; at most 1024 experts, 32 a token.  Logits are float32.
    A token with a NaN or +inf among its logits has weights of NaN."""
    pair = native.route_tokens(x, router, top_k, normalize)
    if pair is not None:
        return pair
    require_cuda(x, 'x')
    require_cuda(router, 'router')
    if x.dtype not in FLOAT_CODES or x.dim() < 1:
        raise ValueError('route_tokens expects float16, bfloat16 or float32 tokens [..., hidden], got {} {}'.format(x.dtype, list(x.shape)))
    if router.dim() != 2 or router.shape[1] != x.shape[-1] or router.dtype not in (x.dtype, torch.float32) or router.device != x.device:
        raise ValueError('expect a router [experts, {}] of {} or float32 on {}, got {} {} on {}'.format(x.shape[-1], x.dtype, x.device, router.dtype, list(router.shape), router.device))
    count = router.shape[0]
    if count > MOST_EXPERTS:
        raise ValueError('{} experts: up to {} are supported'.format(count, MOST_EXPERTS))
    if not isinstance(top_k, int) or isinstance(top_k, bool) or not 1 <= top_k <= min(MOST_TOP, count):
        raise ValueError('top_k must be a whole number of 1 to {}, got {!r}'.format(min(MOST_TOP, count), top_k))
    rows, router = lines_of(rows_of(x)), router.contiguous()
    experts = torch.empty(list(x.shape[:-1]) + [top_k], dtype=torch.int32, device=x.device)
    weights = torch.empty(list(x.shape[:-1]) + [top_k], dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        ffi.func('b200q_route_tokens')(rows.data_ptr(), rows.stride(0), router.data_ptr(), experts.data_ptr(), weights.data_ptr(), rows.shape[0], rows.shape[1], count, top_k,
                                       int(not normalize), FLOAT_CODES[x.dtype], FLOAT_CODES[router.dtype], current_stream_ptr(x.device))
    return experts, weights


def mixture_of_experts(x: torch.Tensor, experts: torch.Tensor, weights: torch.Tensor, gate_up: torch.Tensor, gate_up_scale: torch.Tensor, down: torch.Tensor,
                       down_scale: torch.Tensor, residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t] = residual[t] + sum_j weights[t, j] * (down[e] h) * down_scale[e] with h = silu(g) * u, (g, u) = (gate_up[e] x[t]) * gate_up_scale[e], e = experts[t, j].

    x [..., hidden] float16 or bfloat16; experts int32 and weights float32 [..., k] (route_tokens, or any other choice: an expert may come twice).
    gate_up int8 [count, 2 inner, hidden], rows 2 f and 2 f + 1 the gate and the up projection's f-th; down int8 [count, hidden, inner]; scales [count, 2 inner] and [count, hidden] of one type (float16,
    bfloat16 or float32).  Negative experts are passed over (padding: a token of nothing but these is its residual, or zeros); one beyond the layer's is passed over and reported by b200q_check_status.
    Rows of x and h are multiplied as whole numbers against their largest element, an element held to 2^-22 of it (float32 elsewhere, and where sizes or bases are no multiples of 16 bytes'
    worth or there are more than 512 experts); the sums of these products are exact, what follows is float32, the result is rounded once and is the same on every run.  That shows only in an output
    that takes next to nothing from an element over 2^10 (f16; 2^12 bf16) times the others'.  out: a contiguous tensor for the result, which may be the residual, or x.

    A few tokens are a stream of the weights of the experts that have one; many (more than 64, or dozens an expert) are matrix products over the tokens sorted by expert, with up to half a gigabyte of
    scratch.  Not differentiable."""
    result = native.experts(x, experts, weights, gate_up, gate_up_scale, down, down_scale, residual, out)
    if result is not None:
        return result
    tensors = ((x, 'x'), (experts, 'experts'), (weights, 'weights'), (gate_up, 'gate_up'), (gate_up_scale, 'gate_up_scale'), (down, 'down'), (down_scale, 'down_scale'),
               (residual, 'residual'), (out, 'out'))
    for t, name in tensors:
        if t is not None:
            require_cuda(t, name)
            if t.device != x.device:
                raise ValueError('{} is on {}, x on {}'.format(name, t.device, x.device))
    if x.dtype not in (torch.float16, torch.bfloat16) or x.dim() < 1:
        raise ValueError('mixture_of_experts expects float16 or bfloat16 tokens [..., hidden], got {} {}'.format(x.dtype, list(x.shape)))
    lead, hidden = list(x.shape[:-1]), x.shape[-1]
    if experts.dtype != torch.int32 or experts.dim() != x.dim() or list(experts.shape[:-1]) != lead:
        raise ValueError('expect int32 experts {} + [k], got {} {}'.format(lead, experts.dtype, list(experts.shape)))
    if weights.dtype != torch.float32 or weights.shape != experts.shape:
        raise ValueError('expect float32 weights {}, got {} {}'.format(list(experts.shape), weights.dtype, list(weights.shape)))
    if gate_up.dtype != torch.int8 or gate_up.dim() != 3 or gate_up.shape[1] % 2 != 0 or gate_up.shape[2] != hidden:
        raise ValueError('expect int8 gate_up [experts, 2 inner, {}], got {} {}'.format(hidden, gate_up.dtype, list(gate_up.shape)))
    count, inner = gate_up.shape[0], gate_up.shape[1] // 2
    if down.dtype != torch.int8 or list(down.shape) != [count, hidden, inner]:
        raise ValueError('expect int8 down {}, got {} {}'.format([count, hidden, inner], down.dtype, list(down.shape)))
    if gate_up_scale.dtype not in FLOAT_CODES or down_scale.dtype != gate_up_scale.dtype or list(gate_up_scale.shape) != [count, 2 * inner] or list(down_scale.shape) != [count, hidden]:
        raise ValueError('expect scales {} and {} of one type, got {} {} and {} {}'.format([count, 2 * inner], [count, hidden], gate_up_scale.dtype, list(gate_up_scale.shape),
                                                                                        down_scale.dtype, list(down_scale.shape)))
    if residual is not None and (residual.dtype != x.dtype or residual.shape != x.shape):
        raise ValueError('expect a residual of {} {}, got {} {}'.format(x.dtype, list(x.shape), residual.dtype, list(residual.shape)))
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out.dtype != x.dtype or out.shape != x.shape or not out.is_contiguous():
        raise ValueError('out must be a contiguous tensor of {} {}'.format(x.dtype, list(x.shape)))
    rows = lines_of(rows_of(x))
    others = rows_of(residual) if residual is not None else None
    experts, weights, gate_up, down = experts.contiguous(), weights.contiguous(), gate_up.contiguous(), down.contiguous()
    gate_up_scale, down_scale = gate_up_scale.contiguous(), down_scale.contiguous()
    with torch.cuda.device(x.device):
        ws_ptr, ws_size = workspaces.get(x.device, ffi.func('b200q_mixture_of_experts_workspace_bytes')(rows.shape[0], hidden, inner, count, experts.shape[-1]))
        ffi.func('b200q_mixture_of_experts')(
            rows.data_ptr(), rows.stride(0), experts.data_ptr(), weights.data_ptr(), gate_up.data_ptr(), gate_up_scale.data_ptr(), down.data_ptr(), down_scale.data_ptr(),
            others.data_ptr() if others is not None else None, others.stride(0) if others is not None else 0, out.data_ptr(), rows.shape[0], hidden, inner, count,
            experts.shape[-1], FLOAT_CODES[x.dtype], FLOAT_CODES[gate_up_scale.dtype], ws_ptr, ws_size, current_stream_ptr(x.device))
    return out
