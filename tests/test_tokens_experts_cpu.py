"""What the linears on int8 tokens and the layers of experts refuse before they touch a GPU."""
import ctypes

import pytest
import torch

import hidet_b200
from hidet_b200 import ffi
from hidet_b200.ffi import ACT_SILU_MUL, BF16, F16, F32, Epilogue

AT = 4096  # an address that nothing is read from: every call here is refused, or has no tokens


def tokens(x=AT, stride=64, norm=None, eps=1e-6, codes=AT, scales=AT, rows=2, width=64, type=F16):
    return ffi.func('b200q_quantize_tokens')(x, stride, norm, eps, codes, scales, rows, width, type, None)


def product(a=AT, a_scale=AT, w=AT, scale=AT, c=AT, m=2, n=64, k=64, layout=0, scale_type=F16, out_type=F16, epilogue=None, **of_epilogue):
    if of_epilogue:
        epilogue = ctypes.byref(Epilogue(**dict(dict(bias=None, residual=None, ldr=0, activation=0), **of_epilogue)))
    return ffi.func('b200q_qlinear_i8_i8')(a, a_scale, w, scale, c, m, n, k, layout, scale_type, out_type, epilogue, None)


def route(x=AT, stride=64, router=AT, experts=AT, weights=AT, tokens=2, width=64, count=8, top=2, over_all=0, type=F16, router_type=F16):
    return ffi.func('b200q_route_tokens')(x, stride, router, experts, weights, tokens, width, count, top, over_all, type, router_type, None)


def experts(x=AT, stride=64, chosen=AT, weights=AT, gate_up=AT, s1=AT, down=AT, s2=AT, residual=None, residual_stride=0, out=AT, tokens=2, hidden=64, inner=32, count=8, top=2, type=F16,
            scale_type=F16, workspace=AT, nbytes=1 << 30):
    return ffi.func('b200q_mixture_of_experts')(x, stride, chosen, weights, gate_up, s1, down, s2, residual, residual_stride, out, tokens, hidden, inner, count, top, type, scale_type, workspace,
                                                nbytes, None)


REFUSALS = [
    (tokens, dict(rows=-1), 'negative'), (tokens, dict(width=-1), 'negative'), (tokens, dict(type=3), 'type'), (tokens, dict(eps=-1.0), 'eps'), (tokens, dict(eps=float('nan')), 'eps'),
    (tokens, dict(x=None), 'null'), (tokens, dict(codes=None), 'null'), (tokens, dict(scales=None), 'null'), (tokens, dict(rows=1 << 40), 'rows'), (tokens, dict(width=1 << 40), 'elements'),
    (tokens, dict(stride=-1), 'stride'),
    (product, dict(m=-1), 'negative'), (product, dict(k=-1), 'negative'), (product, dict(layout=2), 'layout'), (product, dict(scale_type=5), 'scales'), (product, dict(out_type=F32), 'f16 or bf16'),
    (product, dict(k=131072), '131071'), (product, dict(m=1 << 40), '2^31'), (product, dict(a=None), 'null'), (product, dict(a_scale=None), 'null'), (product, dict(w=None), 'null'),
    (product, dict(scale=None), 'null'), (product, dict(c=None), 'null'), (product, dict(activation=4), 'activation'), (product, dict(activation=ACT_SILU_MUL, n=63), 'even'),
    (product, dict(residual=AT, ldr=63), 'shorter'),
    (route, dict(tokens=-1), 'negative'), (route, dict(type=4), 'type'), (route, dict(router_type=BF16), 'router'), (route, dict(count=1025), '1024'), (route, dict(top=0), 'experts'),
    (route, dict(top=9), 'experts'), (route, dict(count=64, top=33), '32'), (route, dict(stride=-1), 'stride'), (route, dict(x=None), 'null'), (route, dict(router=None), 'null'),
    (route, dict(experts=None), 'null'), (route, dict(weights=None), 'null'), (route, dict(tokens=1 << 40), 'tokens'),
    (experts, dict(tokens=-1), 'negative'), (experts, dict(stride=-1), 'stride'), (experts, dict(residual_stride=-1), 'stride'), (experts, dict(type=F32), 'f16 or bf16'), (experts, dict(scale_type=3), 'scales'),
    (experts, dict(tokens=1 << 30), 'tokens'), (experts, dict(inner=1 << 30), 'tokens'), (experts, dict(x=None), 'null'), (experts, dict(out=None), 'null'), (experts, dict(chosen=None), 'null'),
    (experts, dict(weights=None), 'null'), (experts, dict(gate_up=None), 'null'), (experts, dict(s1=None), 'null'), (experts, dict(down=None), 'null'), (experts, dict(s2=None), 'null'),
    (experts, dict(workspace=None), 'workspace'), (experts, dict(nbytes=100), 'workspace'),
]


@pytest.mark.parametrize('call,changed,text', REFUSALS)
def test_the_library_refuses(call, changed, text):
    with pytest.raises(ffi.BackendException, match=text.replace('^', '\\^')):
        call(**changed)


def test_nothing_to_do_is_no_launch():
    assert tokens(rows=0) == ffi.OK and product(m=0) == ffi.OK and product(n=0) == ffi.OK and route(tokens=0) == ffi.OK and experts(tokens=0) == ffi.OK


def test_tensors_on_the_cpu_are_refused():
    x, codes = torch.zeros(2, 32, dtype=torch.float16), torch.zeros(2, 32, dtype=torch.int8)
    one = torch.ones(2)
    for call in (lambda: hidet_b200.quantize_tokens(x), lambda: hidet_b200.symmetric_quant_matmul_i8(codes, one, torch.zeros(32, 16, dtype=torch.int8), torch.ones(16)),
                 lambda: hidet_b200.route_tokens(x, torch.zeros(4, 32, dtype=torch.float16), 2),
                 lambda: hidet_b200.mixture_of_experts(x, torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, 1), torch.zeros(4, 64, 32, dtype=torch.int8), torch.ones(4, 64),
                                                       torch.zeros(4, 32, 32, dtype=torch.int8), torch.ones(4, 32))):
        with pytest.raises(ffi.BackendException, match='CUDA'):
            call()


def test_workspace_of_experts():
    need = ffi.func('b200q_mixture_of_experts_workspace_bytes')
    assert need(0, 64, 64, 8, 2) == 0
    assert 0 < need(1, 4096, 14336, 8, 2) <= need(64, 4096, 14336, 8, 2)


@pytest.mark.parametrize('tokens,hidden,inner,count,top', [(2048, 4096, 14336, 8, 2), (10 ** 6, 4096, 14336, 8, 2), (1000, 131056, 16, 512, 1), (4096, 2048, 768, 128, 8), (300, 16, 16, 1, 1), (10 ** 7, 8192, 28672, 512, 8)])
def test_scratch_of_many_tokens_is_bounded(tokens, hidden, inner, count, top):
    need = ffi.func('b200q_mixture_of_experts_workspace_bytes')
    assert 0 < need(65, hidden, inner, count, top) and need(tokens, hidden, inner, count, top) <= 1 << 29
