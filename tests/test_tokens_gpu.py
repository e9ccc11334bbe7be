"""Quantization of tokens and the int8 x int8 product against plain 64-bit forms (token_reference.py)."""
import pytest
import torch

import hidet_b200
import token_reference as ref
from hidet_b200 import ffi

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def generator(*seed):
    return torch.Generator(device='cuda').manual_seed(hash(seed) % (1 << 31))


def normal(gen, *shape, dtype=F32, std=1.0):
    return (torch.randn(shape, generator=gen, device='cuda') * std).to(dtype)


def codes_of(gen, *shape):
    return torch.randint(-127, 128, shape, generator=gen, device='cuda', dtype=torch.int8)


# ---- quantize_tokens ----

def check_tokens(x, norm=None, eps=1e-6):
    codes, scales = hidet_b200.quantize_tokens(x, norm, eps)
    assert codes.shape == x.shape and codes.dtype == torch.int8 and scales.shape == x.shape[:-1] and scales.dtype == F32
    exact, want = ref.quantized(x, norm, eps)
    # the product with the norm, the quotient 127 / amax and the product with it: three roundings of at most 127, then a rounding to whole numbers
    assert (codes.double() - exact).abs().max() <= 0.5 + 127 * 4 * 2.0 ** -24
    # a sum of squares in parts of at most 64 elements a thread and 10 additions, a quotient, a sum, a root, two quotients; the root halves what is in front of it
    n = 8 if norm is None else 8 + (64 + 16) / 2
    assert torch.all((scales.double() - want).abs() <= want * n * 2.0 ** -24 + 2.0 ** -150)
    if x.shape[-1] and norm is None:
        assert torch.all(codes.abs().amax(-1) == torch.where(x.float().abs().amax(-1) > 0, 127, 0))


@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('rows,width', [(1, 1), (3, 7), (5, 8), (2, 255), (7, 1000), (33, 2048), (4, 4096), (3, 11008), (2, 16400), (2, 32768), (2, 40004), (1000, 64)])
def test_quantize_tokens(rows, width, dtype):
    gen = generator(rows, width)
    x = normal(gen, rows, width, dtype=dtype)
    norm = (1 + normal(gen, width, std=0.2)).to(dtype)
    check_tokens(x)
    check_tokens(x, norm, 1e-5)


@pytest.mark.parametrize('dtype', [F16, BF16, F32])
@pytest.mark.parametrize('width', [200, 1536, 5000, 20000])
def test_quantize_tokens_is_the_formula_in_float(width, dtype):
    """Bit for bit, also where products lie in the middle between whole numbers: rows whose largest element is 127 times a small number, of multiples of half of that."""
    gen = generator(1, width)
    x = normal(gen, 64, width, dtype=F32)
    small = torch.arange(1, 33, device='cuda').float()[:, None] * 2.0 ** -12
    x[:32] = (torch.randint(-127, 127, (32, width), generator=gen, device='cuda') + 0.5) * small
    x[:32, 7] = 127 * small[:, 0]
    x = x.to(dtype)
    amax = x.float().abs().amax(-1, keepdim=True)
    codes, scales = hidet_b200.quantize_tokens(x)
    assert torch.equal(codes, torch.round(x.float() * (torch.full_like(amax, 127.0) / amax)).to(torch.int8))
    assert torch.equal(scales, (amax / torch.full_like(amax, 127.0))[:, 0])
    norm = (1 + normal(gen, width, std=0.2)).to(dtype)
    y = x.float() * norm.float()
    amax = y.abs().amax(-1, keepdim=True)
    assert torch.equal(hidet_b200.quantize_tokens(x, norm)[0], torch.round(y * (torch.full_like(amax, 127.0) / amax)).to(torch.int8))
    ones = torch.ones_like(norm)
    assert torch.equal(hidet_b200.quantize_tokens(x, ones)[0], codes)


def test_quantize_tokens_of_any_strides_and_shapes():
    gen = generator(2)
    big = normal(gen, 3, 5, 700, dtype=F16)
    for x in (big[:, :, :640], big[:, :, 1:641], big[:, 1:4, 3:], big.transpose(0, 1), big[..., ::2], big[0, 0], big[:, :1].expand(3, 5, 700), big[:, :, :0].transpose(0, 1)):
        want = hidet_b200.quantize_tokens(x.contiguous())
        got = hidet_b200.quantize_tokens(x)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[0].shape == x.shape
    for shape in ((0, 16), (4, 0), (2, 0, 8)):
        codes, scales = hidet_b200.quantize_tokens(torch.zeros(shape, dtype=F16, device='cuda'))
        assert list(codes.shape) == list(shape) and not scales.any()


@pytest.mark.parametrize('normed', [False, True])
def test_quantize_tokens_of_rows_that_are_no_numbers(normed):
    norm = torch.ones(300, dtype=F32, device='cuda') if normed else None
    x = normal(generator(3), 8, 300)
    x[1, 5], x[2, 299], x[3, 0] = float('nan'), float('inf'), -float('inf')
    x[4] = 0
    x[5] *= 2.0 ** -110
    codes, scales = hidet_b200.quantize_tokens(x, norm, 1e-6)
    assert scales[1:4].isnan().all() and not codes[1:6].any() and not scales[4:6].any()
    ok = [0, 6, 7]
    clean = hidet_b200.quantize_tokens(x[ok].contiguous(), norm, 1e-6)
    assert torch.equal(codes[ok], clean[0]) and torch.equal(scales[ok], clean[1])
    if normed:
        x[6] *= 1e25  # squares beyond float
        assert hidet_b200.quantize_tokens(x, norm, 1e-6)[1][6].isnan()
    else:
        x[6] *= 1e35
        check_tokens(x[6:7])


# ---- the product ----

def check_product(m, k, n, layout='KN', dtype=F16, scale_dtype=F16, bias=False, residual=False, pairs=False, seed=0):
    gen = generator(m, k, n, seed)
    a, w = codes_of(gen, m, k), codes_of(gen, *((k, n) if layout == 'KN' else (n, k)))
    a_scale = normal(gen, m).abs() * 0.02
    scale = (normal(gen, n).abs() * 0.001 + 1e-4).to(scale_dtype)
    b = normal(gen, n, dtype=dtype) if bias else None
    r = normal(gen, m, n // 2 if pairs else n, dtype=dtype) if residual else None
    c = hidet_b200.symmetric_quant_matmul_i8(a, a_scale, w, scale, weight_layout=layout, bias=b, residual=r, activation='silu_mul' if pairs else None, dtype=dtype)
    want, bound = ref.product(a, a_scale, w, scale, layout, b, r, pairs, dtype)
    # beyond the type's largest number the nearest is infinity
    most = torch.finfo(dtype).max
    inside = want.abs() + bound < most
    ref.check(torch.where(inside, c.double(), 0.0), torch.where(inside, want, 0.0), bound)


ROWS = [1, 2, 7, 16, 17, 32, 33, 64, 65, 96, 128, 129, 200, 257, 333, 512, 1000]


@pytest.mark.parametrize('layout', ['KN', 'NK'])
@pytest.mark.parametrize('m', ROWS)
def test_product_by_rows(m, layout):
    check_product(m, 1040, 784, layout)
    check_product(m, 256, 1536, layout, BF16, bias=True, residual=True)
    check_product(m, 528, 544, layout, pairs=True, bias=m % 2 == 0)


@pytest.mark.parametrize('layout', ['KN', 'NK'])
@pytest.mark.parametrize('k,n', [(16, 16), (32, 48), (112, 128), (128, 144), (144, 1040), (2000, 256), (4096, 64), (8208, 272), (12304, 2064), (64, 30000)])
def test_product_by_sizes(k, n, layout):
    for m in (1, 20, 70, 300):
        check_product(m, k, n, layout, pairs=n % 32 == 0)
        check_product(m, k, n, layout, BF16, F32, residual=True)


@pytest.mark.parametrize('layout', ['KN', 'NK'])
@pytest.mark.parametrize('m,k,n', [(606, 2720, 16), (700, 8192, 512), (685, 4016, 16), (500, 8208, 784), (990, 16384, 272), (1, 656, 4880), (1, 992, 16), (121, 8208, 2064), (40, 4096, 6160), (2500, 512, 1040)])
def test_product_whose_inner_dimension_is_shared(m, k, n, layout):
    """Sizes for which CTAs or pairs of them share K by one, two, four and eight."""
    check_product(m, k, n, layout, bias=True, residual=True)
    check_product(m, k, n, layout, BF16, pairs=True)


@pytest.mark.parametrize('layout', ['KN', 'NK'])
@pytest.mark.parametrize('m,k,n', [(1, 1, 1), (3, 5, 7), (2, 130, 66), (70, 513, 131), (65, 64, 100), (9, 1000, 24), (130, 24, 40), (5, 4100, 18)])
def test_product_of_any_alignment(m, k, n, layout):
    check_product(m, k, n, layout, bias=True, residual=True)
    check_product(m, k, n, layout, BF16, BF16, pairs=n % 2 == 0)


def test_product_of_unaligned_bases_and_strided_operands():
    gen = generator(4)
    a, w = codes_of(gen, 40 * 256 + 1)[1:].view(40, 256), codes_of(gen, 256 * 128 + 3)[3:].view(256, 128)
    a_scale, scale = normal(gen, 40).abs(), normal(gen, 128, dtype=F16).abs()
    want = hidet_b200.symmetric_quant_matmul_i8(a.clone(), a_scale, w.clone(), scale)
    for got in (hidet_b200.symmetric_quant_matmul_i8(a, a_scale, w, scale), hidet_b200.symmetric_quant_matmul_i8(a, a_scale, w.clone(), scale),
                hidet_b200.symmetric_quant_matmul_i8(a.clone(), a_scale, w.t().contiguous(), scale, weight_layout='NK'),
                hidet_b200.symmetric_quant_matmul_i8(a.t().contiguous().t(), a_scale, w.t().contiguous().t(), scale),
                hidet_b200.symmetric_quant_matmul_i8(a.view(2, 4, 5, 256), a_scale.view(2, 4, 5), w, scale).view(40, 128)):
        assert torch.equal(got, want)
    out = torch.empty(40 * 128 + 1, dtype=F16, device='cuda')[1:].view(40, 128)
    assert torch.equal(hidet_b200.symmetric_quant_matmul_i8(a, a_scale, w, scale, out=out), want)


def test_product_of_nothing():
    one = torch.ones(0, dtype=F32, device='cuda')
    w, scale = torch.zeros(32, 48, dtype=torch.int8, device='cuda'), torch.ones(48, dtype=F16, device='cuda')
    assert hidet_b200.symmetric_quant_matmul_i8(torch.zeros(0, 32, dtype=torch.int8, device='cuda'), one, w, scale).shape == (0, 48)
    bias = torch.arange(48, device='cuda').half()
    none = hidet_b200.symmetric_quant_matmul_i8(torch.zeros(5, 0, dtype=torch.int8, device='cuda'), torch.ones(5, device='cuda'), w[:0], scale, bias=bias)
    assert torch.equal(none, bias.expand(5, 48))


@pytest.mark.parametrize('layout', ['KN', 'NK'])
@pytest.mark.parametrize('m', [3, 200])
def test_product_of_the_largest_sums(m, layout):
    """The longest rows of the largest codes: 131071 * 2^14 is the last sum that 32 bits hold."""
    k, n = 131056, 32
    a, w = torch.full((m, k), -128, dtype=torch.int8, device='cuda'), torch.full((k, n) if layout == 'KN' else (n, k), -128, dtype=torch.int8, device='cuda')
    scale = torch.full((m,), 2.0 ** -31, device='cuda')
    c = hidet_b200.symmetric_quant_matmul_i8(a, scale, w, torch.ones(n, device='cuda'), weight_layout=layout)
    assert torch.all(c == torch.tensor(k * 2.0 ** -17).half().cuda())
    c = hidet_b200.symmetric_quant_matmul_i8(torch.full((2, 131071), 127, dtype=torch.int8, device='cuda'), scale[:2], torch.full((131071, 3), -128, dtype=torch.int8, device='cuda'),
                                             torch.ones(3, device='cuda'))
    assert torch.all(c == torch.tensor(-131071 * 127 * 2.0 ** -24).half().cuda())


def test_rows_do_not_touch_one_another():
    """A row of NaN, and rows behind the last, leave the others' bits as they are; a row's result does not depend on how many there are beside it, up to the kernel's sums, which are exact."""
    gen = generator(5)
    x, w = normal(gen, 300, 512, dtype=F16), normal(gen, 512, 256, dtype=F16, std=0.02)
    wq, scale = hidet_b200.symmetric_quantize(w, 'int8', dims=0)
    clean = hidet_b200.symmetric_quant_matmul_i8(*hidet_b200.quantize_tokens(x), wq, scale)
    x[7, 3] = float('nan')
    got = hidet_b200.symmetric_quant_matmul_i8(*hidet_b200.quantize_tokens(x), wq, scale)
    assert got[7].isnan().all()
    keep = torch.arange(300, device='cuda') != 7
    assert torch.equal(got[keep], clean[keep])
    for m in (1, 5, 17, 40, 100, 290):
        codes, scales = hidet_b200.quantize_tokens(x[10:10 + m])
        out = torch.full((m + 1, 256), 5.0, dtype=F16, device='cuda')
        hidet_b200.symmetric_quant_matmul_i8(codes, scales, wq, scale, out=out[:m])
        assert torch.equal(out[:m], clean[10:10 + m]) and torch.all(out[m] == 5)


@pytest.mark.parametrize('m', [2, 40, 300])
def test_the_result_may_take_the_residual_s_place(m):
    gen = generator(6, m)
    a, w = codes_of(gen, m, 512), codes_of(gen, 512, 400)
    a_scale, scale, r = normal(gen, m).abs() * 0.01, normal(gen, 400, dtype=F16).abs() * 0.01, normal(gen, m, 400, dtype=F16)
    want = hidet_b200.symmetric_quant_matmul_i8(a, a_scale, w, scale, residual=r)
    assert torch.equal(hidet_b200.symmetric_quant_matmul_i8(a, a_scale, w, scale, residual=r, out=r), want) and torch.equal(r, want)


def test_tokens_and_product_captured_and_on_another_stream():
    gen = generator(7)
    x = normal(gen, 48, 1024, dtype=BF16)
    norm = (1 + normal(gen, 1024, std=0.1)).to(BF16)
    wq, scale = hidet_b200.symmetric_quantize(normal(gen, 2048, 1024, dtype=BF16, std=0.02), 'int8', dims=-1)

    def step():
        return hidet_b200.symmetric_quant_matmul_i8(*hidet_b200.quantize_tokens(x, norm), wq, scale, weight_layout='NK', activation='silu_mul', dtype=BF16)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    other = normal(gen, 48, 1024, dtype=BF16)
    for values in (other, x.clone()):
        x.copy_(values)
        graph.replay()
        assert torch.equal(out, step())
    assert ffi.func('b200q_check_status')() == ffi.OK


def test_refusals():
    a, s = torch.zeros(2, 32, dtype=torch.int8, device='cuda'), torch.ones(2, device='cuda')
    w, scale = torch.zeros(32, 48, dtype=torch.int8, device='cuda'), torch.ones(48, dtype=F16, device='cuda')
    x = torch.zeros(2, 32, dtype=F16, device='cuda')
    f = hidet_b200.symmetric_quant_matmul_i8
    for call, text in ((lambda: hidet_b200.quantize_tokens(a), 'float16'), (lambda: hidet_b200.quantize_tokens(x, torch.ones(31, dtype=F16, device='cuda')), 'norm'),
                       (lambda: hidet_b200.quantize_tokens(x, torch.ones(32, device='cuda')), 'norm'), (lambda: f(x, s, w, scale), 'int8'), (lambda: f(a, s, w.half(), scale), 'int8'),
                       (lambda: f(a, s, w[:31], scale), '32'), (lambda: f(a, s.half(), w, scale), 'a_scale'), (lambda: f(a, s[:1], w, scale), 'a_scale'), (lambda: f(a, s, w, scale[:47]), 'scale'),
                       (lambda: f(a, s, w, scale.int()), 'scale'), (lambda: f(a, s, w, scale, weight_layout='MN'), 'weight_layout'), (lambda: f(a, s, w, scale, activation='gelu'), 'activation'),
                       (lambda: f(a, s, w, scale, dtype=F32), 'float16 or bfloat16'), (lambda: f(a, s, w[:, :47], scale[:47], activation='silu_mul'), 'pairs'),
                       (lambda: f(a, s, w, scale, bias=torch.zeros(48, device='cuda')), 'bias'), (lambda: f(a, s, w, scale, residual=torch.zeros(2, 47, dtype=F16, device='cuda')), 'residual'),
                       (lambda: f(a, s, w, scale, residual=torch.zeros(2, 48, dtype=F16, device='cuda'), activation='silu_mul'), 'residual'),
                       (lambda: f(a, s, w, scale, out=torch.zeros(48, 2, dtype=F16, device='cuda').t()), 'out'), (lambda: f(a, s, w, scale, out=torch.zeros(2, 48, device='cuda')), 'out'),
                       (lambda: f(torch.zeros(1, 131072, dtype=torch.int8, device='cuda'), s[:1], torch.zeros(131072, 1, dtype=torch.int8, device='cuda'), scale[:1]), '131071')):
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(ffi.BackendException, match='eps'):
        hidet_b200.quantize_tokens(x, eps=-1.0)


# ---- beyond 32 bits ----

def far_rows(gen, rows, width, stride, dtype):
    """Rows that lie `stride` elements apart, in memory of which nothing else is written."""
    x = torch.empty((rows - 1) * stride + width, dtype=dtype, device='cuda').as_strided((rows, width), (stride, 1))
    x.copy_(normal(gen, rows, width, dtype=dtype))
    return x


def test_tokens_far_apart_and_many():
    gen = generator(30)
    x = far_rows(gen, 3, 520, (1 << 30) + 8, BF16)
    codes, scales = hidet_b200.quantize_tokens(x)
    want = hidet_b200.quantize_tokens(x.contiguous())
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
    del x
    x = torch.zeros((1 << 18) + 40, 8192, dtype=BF16, device='cuda')  # more than 2^31 elements
    x[-40:] = normal(gen, 40, 8192, dtype=BF16)
    codes, scales = hidet_b200.quantize_tokens(x)
    want = hidet_b200.quantize_tokens(x[-40:].clone())
    assert torch.equal(codes[-40:], want[0]) and torch.equal(scales[-40:], want[1]) and not scales[:-40].any()


@pytest.mark.parametrize('m,k,n', [((1 << 18) + 40, 8192, 16), ((1 << 17) + 40, 64, 16400), ((1 << 17) + 41, 62, 16402)])
def test_products_of_more_than_32_bits_of_elements(m, k, n):
    gen = generator(31, n)
    a, scales = torch.zeros(m, k, dtype=torch.int8, device='cuda'), torch.ones(m, device='cuda')
    a[-40:] = codes_of(gen, 40, k)
    w, scale = codes_of(gen, k, n), torch.full((n,), 1e-3, device='cuda')
    r = torch.zeros(m, n, dtype=F16, device='cuda')
    r[-40:] = normal(gen, 40, n, dtype=F16)
    added = r[-40:].clone()
    got = hidet_b200.symmetric_quant_matmul_i8(a, scales, w, scale, residual=r, out=r)
    assert not got[:-40].any()
    # the sum is exact; its product with the scale is one rounding, the addition another, the result the last
    want = (a[-40:].double() @ w.double()) * scale.double()
    both = want + added.double()
    assert torch.all((got[-40:].double() - both).abs() <= both.abs() * 2.0 ** -11 + (want.abs() + both.abs()) * 2.0 ** -23 + 2.0 ** -24)
