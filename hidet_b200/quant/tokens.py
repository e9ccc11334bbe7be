"""Linears on int8 tokens: the quantization of tokens, and the int8 x int8 product with a scale for each token and each output channel.

    codes, scales = quantize_tokens(x, norm=weight_of_the_norm)
    y = symmetric_quant_matmul_i8(codes, scales, weight, weight_scale)

weight and weight_scale are symmetric_quantize's, as for symmetric_quant_matmul, whose tokens stay float16: that one is for a few tokens, where reading the weight is all
the time, and this one for many, where int8 products run at twice the rate.  Not offered by the reference.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from .. import ffi, native
from ..runtime import FLOAT_CODES, current_stream_ptr, require_cuda
from .matmul import _ACTIVATIONS, _LAYOUTS

MOST_INNER = 131071  # products of a sum that 32 bits hold


def rows_of(x: torch.Tensor) -> torch.Tensor:
    """x [..., width] as rows [n, width] with neighbouring elements, without a copy where its strides allow that."""
    rows = x.reshape(-1, x.shape[-1]) if x.numel() else x.new_empty((math.prod(x.shape[:-1]), x.shape[-1]))
    return rows if rows.stride(1) == 1 or rows.shape[1] <= 1 else rows.contiguous()


def quantize_tokens(x: torch.Tensor, norm: Optional[torch.Tensor] = None, eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of x [..., width] (float16, bfloat16 or float32): int8 of x's shape and float32 [...].

    A token's code is rint(y * (127 / amax)), its scale amax / 127, amax the largest magnitude of its y: x itself or, with norm [width] (of x's type),
    the RMS norm x / sqrt(mean(x^2) + eps) * norm, which is not rounded in between.  Tokens of zeros (below 2^-100) have a scale of zero; a token with a NaN or an infinity
    (or whose squares are beyond float32 in front of a norm) has a scale of NaN, and so whatever is computed from it is NaN.

    What it returns for rows [N, K] may also be a weight, at once: symmetric_quant_matmul_i8(*quantize_tokens(x), *quantize_tokens(w), weight_layout='NK')."""
    pair = native.quantize_tokens(x, norm, eps)
    if pair is not None:
        return pair
    require_cuda(x, 'x')
    if x.dtype not in FLOAT_CODES or x.dim() < 1:
        raise ValueError('quantize_tokens expects float16, bfloat16 or float32 [..., width], got {} {}'.format(x.dtype, list(x.shape)))
    if norm is not None:
        require_cuda(norm, 'norm')
        if norm.dtype != x.dtype or list(norm.shape) != [x.shape[-1]] or norm.device != x.device:
            raise ValueError('expect a norm of {} [{}] on {}, got {} {} on {}'.format(x.dtype, x.shape[-1], x.device, norm.dtype, list(norm.shape), norm.device))
        norm = norm.contiguous()
    rows = rows_of(x)
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        ffi.func('b200q_quantize_tokens')(rows.data_ptr(), rows.stride(0), norm.data_ptr() if norm is not None else None, eps, codes.data_ptr(), scales.data_ptr(),
                                          rows.shape[0], rows.shape[1], FLOAT_CODES[x.dtype], current_stream_ptr(x.device))
    return codes, scales


def symmetric_quant_matmul_i8(a: torch.Tensor, a_scale: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, weight_layout: str = 'KN',
                              out: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                              activation: Optional[str] = None, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """c[..., M, N] = (a[..., M, K] @ weight) * scale * a_scale[..., M, None] in `dtype` (float16 or bfloat16).

    a int8 with a_scale float32 (quantize_tokens), weight int8 [K, N] (weight_layout 'KN') or [N, K] ('NK') with scale [N] (float16, bfloat16 or float32).
    Every operand may be the result of the call in front.  The sum over k is exact (K up to 131071); scales, bias [N], activation and residual (both of `dtype`, in symmetric_quant_matmul's order and meaning, for either layout)
    are float and the result is rounded once.  out: a contiguous tensor for the result, which may be the residual."""
    c = native.matmul_i8(a, a_scale, weight, scale, weight_layout, out, bias, residual, activation, dtype)
    if c is not None:
        return c
    for t, name in ((a, 'a'), (a_scale, 'a_scale'), (weight, 'weight'), (scale, 'scale'), (bias, 'bias'), (residual, 'residual'), (out, 'out')):
        if t is not None:
            require_cuda(t, name)
            if t.device != a.device:
                raise ValueError('{} is on {}, a on {}'.format(name, t.device, a.device))
    if weight_layout not in _LAYOUTS:
        raise ValueError("weight_layout must be 'KN' or 'NK', got {!r}".format(weight_layout))
    if activation not in _ACTIVATIONS:
        raise ValueError("activation must be None or 'silu_mul', got {!r}".format(activation))
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError('results are float16 or bfloat16, not {}'.format(dtype))
    if a.dtype != torch.int8 or weight.dtype != torch.int8 or a.dim() < 1 or weight.dim() != 2:
        raise ValueError('expect int8 tokens [..., K] and an int8 weight of two dimensions, got {} {} and {} {}'.format(a.dtype, list(a.shape), weight.dtype, list(weight.shape)))
    k, n = weight.shape if weight_layout == 'KN' else weight.shape[::-1]
    if a.shape[-1] != k:
        raise ValueError('tokens of {} elements for a weight of {}'.format(a.shape[-1], k))
    if k > MOST_INNER:
        raise ValueError('sums of {} products: up to {} fit 32 bits'.format(k, MOST_INNER))
    if a_scale.dtype != torch.float32 or a_scale.shape != a.shape[:-1]:
        raise ValueError('expect float32 a_scale {}, got {} {}'.format(list(a.shape[:-1]), a_scale.dtype, list(a_scale.shape)))
    if scale.dtype not in FLOAT_CODES or list(scale.shape) != [n]:
        raise ValueError('expect a scale of shape [{}], got {} {}'.format(n, scale.dtype, list(scale.shape)))
    pairs = _ACTIVATIONS[activation] == ffi.ACT_SILU_MUL
    if pairs and n % 2 != 0:
        raise ValueError('{} output channels are no pairs'.format(n))
    out_shape = list(a.shape[:-1]) + [n // 2 if pairs else n]
    if bias is not None:
        if bias.dtype != dtype or list(bias.shape) != [n]:
            raise ValueError('expect a bias of {} [{}], got {} {}'.format(dtype, n, bias.dtype, list(bias.shape)))
        bias = bias.contiguous()
    if residual is not None:
        if residual.dtype != dtype or list(residual.shape) != out_shape:
            raise ValueError('expect a residual of {} {}, got {} {}'.format(dtype, out_shape, residual.dtype, list(residual.shape)))
        residual = residual.contiguous()
    if out is None:
        out = torch.empty(out_shape, dtype=dtype, device=a.device)
    elif list(out.shape) != out_shape or out.dtype != dtype or not out.is_contiguous():
        raise ValueError('out must be a contiguous tensor of {} {}'.format(dtype, out_shape))
    a, a_scale, weight, scale = a.contiguous(), a_scale.contiguous(), weight.contiguous(), scale.contiguous()
    epilogue = ffi.Epilogue(bias.data_ptr() if bias is not None else None, residual.data_ptr() if residual is not None else None, out_shape[-1], _ACTIVATIONS[activation])
    with torch.cuda.device(a.device):
        ffi.func('b200q_qlinear_i8_i8')(a.data_ptr(), a_scale.data_ptr(), weight.data_ptr(), scale.data_ptr(), out.data_ptr(), a_scale.numel(), n, k, _LAYOUTS[weight_layout],
                                        FLOAT_CODES[scale.dtype], FLOAT_CODES[dtype], ctypes.byref(epilogue), current_stream_ptr(a.device))
    return out
