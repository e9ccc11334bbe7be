"""csrc/host.cpp's part of the linears on int8 tokens and the layers of experts: the same results as the Python paths, None for what it does not serve."""
import pytest
import torch

import hidet_b200
from hidet_b200 import native
from test_experts_gpu import choices, layer
from test_native_gpu import _both
from test_tokens_gpu import BF16, F16, F32, codes_of, generator, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def loaded():
    assert native.load() is not None


@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('shape', [(1, 256), (3, 5, 77), (4096,)])
def test_quantize_tokens(monkeypatch, shape, dtype):
    gen = generator(31, len(shape))
    x, norm = normal(gen, *shape, dtype=dtype), normal(gen, shape[-1], dtype=dtype)
    for w in (None, norm):
        _both(monkeypatch, 'quantize_tokens', (x, w, 1e-5), lambda: hidet_b200.quantize_tokens(x, w, 1e-5))


@pytest.mark.parametrize('layout', ['KN', 'NK'])
@pytest.mark.parametrize('lead', [(1,), (2, 9), (300,)])
def test_product(monkeypatch, lead, layout):
    gen = generator(32, len(lead))
    a, w = codes_of(gen, *lead, 256), codes_of(gen, *((256, 96) if layout == 'KN' else (96, 256)))
    a_scale, scale = normal(gen, *lead), normal(gen, 96, dtype=BF16)
    for dtype in (F16, BF16):
        bias, residual, half = normal(gen, 96, dtype=dtype), normal(gen, *lead, 96, dtype=dtype), normal(gen, *lead, 48, dtype=dtype)
        out = torch.empty_like(residual)
        for args in ((None, None, None, None), (None, bias, residual, None), (None, None, half, 'silu_mul'), (out, bias, None, None)):
            got = _both(monkeypatch, 'matmul_i8', (a, a_scale, w, scale, layout) + args + (dtype,),
                        lambda: hidet_b200.symmetric_quant_matmul_i8(a, a_scale, w, scale, layout, *args, dtype=dtype))
            assert args[0] is None or got is out


def test_route(monkeypatch):
    gen = generator(33)
    for dtype, router_dtype in ((F16, F16), (BF16, F32), (F32, F32)):
        x, r = normal(gen, 2, 3, 200, dtype=dtype), normal(gen, 12, 200, dtype=router_dtype)
        for normalize in (True, False):
            _both(monkeypatch, 'route_tokens', (x, r, 4, normalize), lambda: hidet_b200.route_tokens(x, r, 4, normalize))


def test_experts(monkeypatch):
    gen = generator(34)
    for dtype, scale_dtype in ((F16, F16), (BF16, F32)):
        x, w = normal(gen, 7, 256, dtype=dtype), layer(gen, 6, 256, 96, scale_dtype)
        chosen, weights = choices(gen, 7, 6, 3)
        hidet_b200.mixture_of_experts(x, chosen, weights, *w)  # makes the stream's scratch
        for residual, out in ((None, None), (x, None), (x, torch.empty_like(x))):
            got = _both(monkeypatch, 'experts', (x, chosen, weights) + w + (residual, out), lambda: hidet_b200.mixture_of_experts(x, chosen, weights, *w, residual=residual, out=out))
            assert out is None or got is out


def test_what_is_not_plain_takes_the_general_path():
    gen = generator(35)
    x, a, w = normal(gen, 4, 64, dtype=F16), codes_of(gen, 4, 64), codes_of(gen, 64, 32)
    s, scale = normal(gen, 4), normal(gen, 32, dtype=F16)
    assert native.quantize_tokens(x, None, 1e-5) is not None
    for args in ((x.t(), None, 1e-5), (x.cpu(), None, 1e-5), (a, None, 1e-5), (x, x[0, :63].contiguous(), 1e-5), (x, x[0].float(), 1e-5), (x, None, 1), (x, None, -1.0), (x[:0], None, 1e-5)):
        assert native.quantize_tokens(*args) is None
    plain = (a, s, w, scale, 'KN', None, None, None, None, F16)
    assert native.matmul_i8(*plain) is not None
    for at, what in ((0, a.t()), (0, x), (1, s.half()), (1, s[:3].contiguous()), (2, w.t()), (2, w[:63].contiguous()), (3, scale[:31].contiguous()), (3, scale.int()), (4, 'NK'), (4, 'MN'), (5, x),
                     (6, scale.float()), (7, x), (8, 'gelu'), (9, F32)):
        assert native.matmul_i8(*(what if i == at else v for i, v in enumerate(plain))) is None, (at, what)
    r = normal(gen, 6, 64, dtype=F16)
    assert native.route_tokens(x, r, 2, True) is not None
    for args in ((x, r, 7, True), (x, r, 0, True), (x, r, 2.0, True), (x, r, 2, 1), (x, r.to(BF16), 2, True), (x, r[:, :63].contiguous(), 2, True), (x[:0], r, 2, True)):
        assert native.route_tokens(*args) is None
    plain = (x, *choices(gen, 4, 6, 2), *layer(gen, 6, 64, 32), None, None)
    hidet_b200.mixture_of_experts(*plain)
    assert native.experts(*plain) is not None
    for at, what in ((0, x.float()), (0, x.t()), (1, plain[1].long()), (1, plain[1][:3].contiguous()), (2, plain[2].half()), (3, plain[3][:5].contiguous()), (4, plain[4].float()), (5, plain[5][:, :, :31].contiguous()),
                     (6, plain[6].int()), (7, x.float()), (8, x.t())):
        assert native.experts(*(what if i == at else v for i, v in enumerate(plain))) is None, (at, what)
