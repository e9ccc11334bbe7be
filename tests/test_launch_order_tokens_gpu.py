"""Operands of the linears on int8 tokens and of the layers of experts that the kernel in front writes, and lets others start before it has: all of them, a weight's codes among them,
are read behind its end.  quantize_tokens is such a kernel itself, and what it returns is a weight."""
import pytest
import torch

import hidet_b200
from hidet_b200 import ffi
from test_launch_order_gpu import _bytes, _check, late_copy, late_copy_everywhere  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def normal(gen, *shape, dtype=F16, std=1.0):
    return torch.randn(*shape, device='cuda', generator=gen).mul_(std).to(dtype)


def codes(gen, *shape):
    return torch.randint(-127, 128, shape, device='cuda', generator=gen, dtype=torch.int8)


def positive(gen, *shape, dtype=F16, size=1e-2):
    return torch.rand(*shape, device='cuda', generator=gen).mul_(size).add_(size / 8).to(dtype)


# a warp a row, a CTA a row, rows that are read twice; whole vectors and others
@pytest.mark.parametrize('rows,width', [(300, 64), (20, 1000), (64, 4096), (400, 4096), (40, 9002), (4, 20000), (2, 40002)])
@pytest.mark.parametrize('dtype', [F16, F32])
@pytest.mark.parametrize('everywhere', [False, True])
def test_tokens_and_norm_are_read_behind_the_kernel_in_front(late_copy, late_copy_everywhere, rows, width, dtype, everywhere):
    gen = torch.Generator(device='cuda').manual_seed(rows + width)
    copy = late_copy_everywhere if everywhere else late_copy
    operands = [(normal(gen, rows, width, dtype=dtype), normal(gen, width, dtype=dtype)) for _ in range(2)]
    _check(copy, operands, lambda x, norm: _bytes(*hidet_b200.quantize_tokens(x, norm=norm)))
    _check(copy, [o[:1] for o in operands], lambda x: _bytes(*hidet_b200.quantize_tokens(x)))


# the kernel for few tokens with and without a cluster, pairs of SMs with a tile each and with a tile's K shared, and the one for any alignment
@pytest.mark.parametrize('m,k,n', [(1, 512, 1024), (4, 4096, 512), (16, 2048, 8192), (100, 1024, 512), (600, 1024, 4096), (1000, 8192, 512), (4, 67, 132), (68, 130, 70)])
@pytest.mark.parametrize('layout', ['KN', 'NK'])
def test_all_operands_of_the_product_are_read_behind_the_kernel_in_front(late_copy, m, k, n, layout):
    gen = torch.Generator(device='cuda').manual_seed(m + k + n)
    operands = [(codes(gen, m, k), positive(gen, m, dtype=F32), codes(gen, *((k, n) if layout == 'KN' else (n, k))), positive(gen, n), normal(gen, n), normal(gen, m, n)) for _ in range(2)]
    _check(late_copy, operands, lambda a, a_scale, w, scale, bias, residual: hidet_b200.symmetric_quant_matmul_i8(a, a_scale, w, scale, weight_layout=layout, bias=bias, residual=residual))


@pytest.mark.parametrize('m,k,n', [(2, 512, 1024), (600, 1024, 4096), (1000, 8192, 512)])
def test_scales_and_weights_may_come_late_on_every_sm(late_copy_everywhere, m, k, n):
    gen = torch.Generator(device='cuda').manual_seed(m + k)
    operands = [(codes(gen, m, k), positive(gen, m, dtype=F32), codes(gen, k, n), positive(gen, n, dtype=F32)) for _ in range(2)]
    _check(late_copy_everywhere, operands, hidet_b200.symmetric_quant_matmul_i8)


@pytest.mark.parametrize('tokens,width,count', [(1, 4096, 8), (7, 2048, 64), (64, 512, 256), (5, 130, 10)])
@pytest.mark.parametrize('dtype,router_dtype', [(F16, F16), (BF16, F32), (F32, F32)])
def test_tokens_and_router_are_read_behind_the_kernel_in_front(late_copy, tokens, width, count, dtype, router_dtype):
    gen = torch.Generator(device='cuda').manual_seed(tokens + width)
    operands = [(normal(gen, tokens, width, dtype=dtype), normal(gen, count, width, dtype=router_dtype, std=width ** -0.5)) for _ in range(2)]
    _check(late_copy, operands, lambda x, router: _bytes(*hidet_b200.route_tokens(x, router, 4)))


# few tokens, many, and kernels for any alignment
@pytest.mark.parametrize('tokens,hidden,inner,count,top', [(1, 512, 768, 8, 2), (16, 512, 256, 4, 2), (200, 512, 256, 8, 2), (3, 200, 36, 4, 2)])
def test_all_operands_of_the_experts_are_read_behind_the_kernel_in_front(late_copy, tokens, hidden, inner, count, top):
    gen = torch.Generator(device='cuda').manual_seed(tokens + hidden)
    operands = [(normal(gen, tokens, hidden), torch.randint(0, count, (tokens, top), device='cuda', generator=gen, dtype=torch.int32), positive(gen, tokens, top, dtype=F32, size=1.0),
                 codes(gen, count, 2 * inner, hidden), positive(gen, count, 2 * inner), codes(gen, count, hidden, inner), positive(gen, count, hidden), normal(gen, tokens, hidden)) for _ in range(2)]
    _check(late_copy, operands, lambda x, e, w, up, s1, down, s2, residual: hidet_b200.mixture_of_experts(x, e, w, up, s1, down, s2, residual=residual))


def quantize_into(x, out, scales):
    ffi.func('b200q_quantize_tokens')(x.data_ptr(), x.shape[1], None, 0.0, out.data_ptr(), scales.data_ptr(), x.shape[0], x.shape[1], ffi.F16, torch.cuda.current_stream().cuda_stream)


# weights of several waves of CTAs
@pytest.mark.parametrize('m,k,n', [(1, 4096, 4096), (3, 4096, 12288), (48, 2048, 8192), (333, 4096, 12288), (1000, 8192, 512), (9, 130, 1000)])
@pytest.mark.parametrize('tokens_first', [False, True])
def test_codes_of_quantize_tokens_are_a_weight_at_once(m, k, n, tokens_first):
    """Over and over into the same memory, which holds another weight's codes until then."""
    gen = torch.Generator(device='cuda').manual_seed(m + n)
    x, weights = normal(gen, m, k), [normal(gen, n, k, std=0.02) for _ in range(2)]
    wq, scale = torch.zeros(n, k, dtype=torch.int8, device='cuda'), torch.zeros(n, device='cuda')
    xq, x_scale = torch.zeros(m, k, dtype=torch.int8, device='cuda'), torch.zeros(m, device='cuda')

    def both(w, between):
        for tokens in ((True, False) if tokens_first else (False, True)):
            quantize_into(*((x, xq, x_scale) if tokens else (w, wq, scale)))
            between()
        return hidet_b200.symmetric_quant_matmul_i8(xq, x_scale, wq, scale, weight_layout='NK')

    want = [both(w, torch.cuda.synchronize) for w in weights]
    torch.cuda.synchronize()
    got = [both(weights[i % 2], lambda: None) for i in range(12)]
    assert not torch.equal(want[0], want[1])
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 2])
    # the same through the package's calls, whose memory the allocator hands round
    for i in range(12):
        w = weights[i % 2]
        first = hidet_b200.quantize_tokens(x) if tokens_first else hidet_b200.quantize_tokens(w)
        second = hidet_b200.quantize_tokens(w) if tokens_first else hidet_b200.quantize_tokens(x)
        a, b = (first, second) if tokens_first else (second, first)
        assert torch.equal(hidet_b200.symmetric_quant_matmul_i8(*a, *b, weight_layout='NK'), want[i % 2])
    assert ffi.func('b200q_check_status')() == ffi.OK


def test_codes_of_quantize_tokens_are_a_weight_at_once_in_a_graph():
    m, k, n = 16, 4096, 8192
    gen = torch.Generator(device='cuda').manual_seed(3)
    x, buffer = normal(gen, m, k), torch.zeros(n, k, dtype=F16, device='cuda')
    weights = [normal(gen, n, k, std=0.02) for _ in range(2)]
    want = [hidet_b200.symmetric_quant_matmul_i8(*hidet_b200.quantize_tokens(x), *[t.clone() for t in hidet_b200.quantize_tokens(w)], weight_layout='NK') for w in weights]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = hidet_b200.symmetric_quant_matmul_i8(*hidet_b200.quantize_tokens(x), *hidet_b200.quantize_tokens(buffer), weight_layout='NK')
    for i in range(8):
        buffer.copy_(weights[i % 2])
        graph.replay()
        assert torch.equal(out, want[i % 2])


# the kernel of f16 rows that reads a weight's first codes ahead of the kernel in front; behind quantize_tokens at once, behind others that let it start early, and captured
@pytest.mark.parametrize('m', [1, 7, 16])
@pytest.mark.parametrize('between', ['nothing', 'tokens', 'route', 'product'])
@pytest.mark.parametrize('captured', [False, True])
def test_codes_of_quantize_tokens_are_a_weight_of_f16_rows_at_once(m, between, captured):
    k, n = 4096, 6144
    gen = torch.Generator(device='cuda').manual_seed(m)
    x, weights = normal(gen, m, k), [normal(gen, n, k, std=0.02) for _ in range(2)]
    scale = torch.full((n,), 1e-3, device='cuda', dtype=F16)   # the caller's own
    w, wq, scales = torch.zeros(n, k, dtype=F16, device='cuda'), torch.zeros(n, k, dtype=torch.int8, device='cuda'), torch.zeros(n, device='cuda')
    router, xq = normal(gen, 8, k, std=0.02), hidet_b200.quantize_tokens(x)
    other, ones = codes(gen, k, 256), torch.ones(256, device='cuda')

    def call(wait):
        quantize_into(w, wq, scales)
        wait()
        if between == 'tokens':
            hidet_b200.quantize_tokens(x)
        elif between == 'route':
            hidet_b200.route_tokens(x, router, 2)
        elif between == 'product':
            hidet_b200.symmetric_quant_matmul_i8(*xq, other, ones)
        return hidet_b200.symmetric_quant_matmul(x, wq, scale, weight_layout='NK')

    want = []
    for source in weights:
        w.copy_(source)
        want.append(call(torch.cuda.synchronize))
    assert not torch.equal(want[0], want[1])
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(lambda: None)
    for i in range(12):
        w.copy_(weights[i % 2])
        if captured:
            graph.replay()
        else:
            out = call(lambda: None)
        assert torch.equal(out, want[i % 2])
    assert ffi.func('b200q_check_status')() == ffi.OK


@pytest.mark.parametrize('tokens', [2, 24, 200])
def test_codes_of_quantize_tokens_are_the_experts_weights_at_once(tokens):
    hidden, inner, count = 1024, 768, 8
    gen = torch.Generator(device='cuda').manual_seed(tokens)
    x, router = normal(gen, tokens, hidden), normal(gen, count, hidden, std=0.05)
    layers = [(normal(gen, count, 2 * inner, hidden, std=0.02), normal(gen, count, hidden, inner, std=0.02)) for _ in range(2)]
    chosen, shares = hidet_b200.route_tokens(x, router, 2)

    def call(up, down, wait):
        up = hidet_b200.quantize_tokens(up)
        wait()
        down = hidet_b200.quantize_tokens(down)
        wait()
        return hidet_b200.mixture_of_experts(x, chosen, shares, *up, *down)

    want = [call(*layer, torch.cuda.synchronize) for layer in layers]
    assert not torch.equal(want[0], want[1])
    for i in range(12):
        assert torch.equal(call(*layers[i % 2], lambda: None), want[i % 2])
    assert ffi.func('b200q_check_status')() == ffi.OK
