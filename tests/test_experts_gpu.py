"""Routing and layers of experts against plain 64-bit forms (token_reference.py)."""
import pytest
import torch

import hidet_b200
import token_reference as ref
from hidet_b200 import ffi
from test_tokens_gpu import BF16, F16, F32, codes_of, far_rows, generator, normal

pytestmark = pytest.mark.gpu


# ---- routing ----

def check_route(x, router, top, normalize=True):
    experts, weights = hidet_b200.route_tokens(x, router, top, normalize)
    assert experts.dtype == torch.int32 and weights.dtype == F32 and list(experts.shape) == list(x.shape[:-1]) + [top] == list(weights.shape)
    logits = x.double() @ router.double().t()
    # float sums in parts of at most width / 32 products a lane, and eight additions
    off = (x.double().abs() @ router.double().abs().t()) * ((x.shape[-1] / 32 + 24) * 2.0 ** -24)
    chosen = logits.gather(-1, experts.long())
    assert torch.all(experts.long().sort(-1)[0].diff(dim=-1) > 0) if top > 1 else True  # no expert twice
    slack = off.amax(-1, keepdim=True)
    assert torch.all(chosen[..., 1:] <= chosen[..., :-1] + 2 * slack)
    rest = logits.scatter(-1, experts.long(), -float('inf')).amax(-1)
    assert torch.all(rest <= chosen[..., -1] + 2 * slack[..., 0])
    p = torch.softmax(logits, -1).gather(-1, experts.long())
    want = p / p.sum(-1, keepdim=True) if normalize else p
    # a change d of every logit changes a share by at most 2 d of itself; the exponential and the quotient are a few roundings, its argument's error (a rounding of a difference) that times the difference
    bound = want * (4 * slack + (16 + (chosen[..., :1] - chosen).abs() + router.shape[0]) * 2.0 ** -23) + 1e-37
    assert torch.all((weights.double() - want).abs() <= bound)


@pytest.mark.parametrize('dtype,router_dtype', [(F16, F16), (BF16, BF16), (F32, F32), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize('tokens,width,count,top', [(1, 512, 8, 2), (3, 1000, 5, 5), (4, 64, 1, 1), (7, 2048, 64, 6), (33, 77, 40, 8), (130, 256, 128, 8), (2, 4096, 1000, 32), (5, 1, 3, 2), (9, 1536, 17, 1)])
def test_route(tokens, width, count, top, dtype, router_dtype):
    gen = generator(tokens, width, count)
    x, router = normal(gen, tokens, width, dtype=dtype), normal(gen, count, width, dtype=router_dtype, std=2 * width ** -0.5)
    check_route(x, router, top)
    check_route(x, router, top, normalize=False)


def test_route_takes_equal_logits_by_index():
    x = torch.ones(5, 32, dtype=F16, device='cuda')
    router = torch.zeros(70, 32, dtype=F16, device='cuda')
    router[[3, 40, 41, 69]] = 1
    router[50] = 2
    experts, weights = hidet_b200.route_tokens(x, router, 7)
    assert experts.tolist() == [[50, 3, 40, 41, 69, 0, 1]] * 5
    assert hidet_b200.route_tokens(x[:, :0], router[:, :0], 3)[0].tolist() == [[0, 1, 2]] * 5


def test_route_of_rows_that_are_no_numbers():
    gen = generator(11)
    x, router = normal(gen, 6, 64), normal(gen, 12, 64)
    x[1, 3], x[2, 5] = float('nan'), float('inf')
    experts, weights = hidet_b200.route_tokens(x, router, 4)
    assert weights[1:3].isnan().all()
    assert torch.all((experts >= 0) & (experts < 12)) and torch.all(experts.sort(-1)[0].diff(dim=-1) > 0)
    ok = [0, 3, 4, 5]
    clean = hidet_b200.route_tokens(x[ok].contiguous(), router, 4)
    assert torch.equal(experts[ok], clean[0]) and torch.equal(weights[ok], clean[1])
    assert hidet_b200.route_tokens(x[:0], router, 4)[0].shape == (0, 4)


def test_route_of_strided_tokens():
    gen = generator(12)
    big, router = normal(gen, 4, 6, 300, dtype=BF16), normal(gen, 16, 256, dtype=BF16)
    for x in (big[..., :256], big[..., 1:257], big.transpose(0, 1)[..., 3:259], big[:, :1, :256].expand(4, 6, 256)):
        got, want = hidet_b200.route_tokens(x, router, 3), hidet_b200.route_tokens(x.contiguous(), router, 3)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- experts ----

def layer(gen, count, hidden, inner, scale_dtype=F16):
    return (codes_of(gen, count, 2 * inner, hidden), (normal(gen, count, 2 * inner).abs() * 2e-4 + 1e-4).to(scale_dtype), codes_of(gen, count, hidden, inner),
            (normal(gen, count, hidden).abs() * 2e-4 + 1e-4).to(scale_dtype))


def choices(gen, tokens, count, top):
    experts = torch.rand((tokens, count), generator=gen, device='cuda').argsort(-1)[:, :top].int().contiguous()
    return experts, torch.rand((tokens, top), generator=gen, device='cuda') + 0.1


def check_layer(x, experts, weights, *w, residual=None):
    got = hidet_b200.mixture_of_experts(x, experts, weights, *w, residual=residual)
    assert got.shape == x.shape and got.dtype == x.dtype
    ref.check(got, *ref.experts(x, experts, weights, *w, residual))
    assert torch.equal(hidet_b200.mixture_of_experts(x, experts, weights, *w, residual=residual), got)  # the same on every run
    return got


@pytest.mark.parametrize('dtype,scale_dtype', [(F16, F16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize('tokens,count,top,hidden,inner', [(1, 8, 2, 512, 1024), (1, 1, 1, 16, 16), (2, 4, 2, 1040, 272), (5, 16, 4, 256, 768), (8, 2, 2, 512, 528), (9, 3, 1, 144, 2064),
                                                         (17, 8, 2, 1024, 512), (33, 64, 6, 512, 176), (64, 4, 2, 256, 512), (64, 2, 2, 1024, 256), (65, 4, 3, 256, 128), (150, 8, 2, 128, 64), (3, 200, 8, 384, 96), (2, 600, 4, 64, 32), (40, 40, 32, 256, 64), (40, 8, 2, 4096, 1024), (6, 8, 2, 2048, 1536)])
def test_layer(tokens, count, top, hidden, inner, dtype, scale_dtype):
    gen = generator(tokens, count, hidden)
    x = normal(gen, tokens, hidden, dtype=dtype)
    check_layer(x, *choices(gen, tokens, count, top), *layer(gen, count, hidden, inner, scale_dtype), residual=normal(gen, tokens, hidden, dtype=dtype) if tokens % 2 else None)


@pytest.mark.parametrize('dtype,scale_dtype', [(F16, F16), (BF16, F32)])
@pytest.mark.parametrize('tokens,count,top,hidden,inner', [(65, 8, 1, 512, 272), (81, 1, 1, 16, 16), (200, 512, 8, 128, 64), (300, 1, 1, 256, 528), (321, 3, 2, 1040, 144), (640, 64, 6, 272, 176), (1000, 8, 2, 2064, 400),
                                                         (100, 40, 32, 144, 256), (4500, 4, 2, 64, 48), (66, 4, 4, 128, 4096), (2000, 2, 1, 256, 128), (70, 600, 2, 64, 32)])
def test_layer_of_many_tokens(tokens, count, top, hidden, inner, dtype, scale_dtype):
    gen = generator(tokens, count, hidden, 1)
    x = normal(gen, tokens, hidden, dtype=dtype)
    experts, weights = choices(gen, tokens, count, top)
    experts[5], experts[-1, 0], experts[7] = -1, -3, experts[7, 0].item()  # nobody's, in part nobody's, one expert for all
    residual = normal(gen, tokens, hidden, dtype=dtype) if tokens % 2 else None
    got = check_layer(x, experts, weights, *layer(gen, count, hidden, inner, scale_dtype), residual=residual)
    assert torch.equal(got[5], residual[5]) if residual is not None else not got[5].any()


@pytest.mark.parametrize('tokens,count,top,hidden,inner', [(1, 3, 2, 50, 30), (7, 4, 2, 129, 65), (70, 2, 1, 24, 8), (2, 2, 2, 1, 1)])
def test_layer_of_any_alignment(tokens, count, top, hidden, inner):
    gen = generator(tokens, hidden)
    check_layer(normal(gen, tokens, hidden, dtype=BF16), *choices(gen, tokens, count, top), *layer(gen, count, hidden, inner), residual=normal(gen, tokens, hidden, dtype=BF16))


@pytest.mark.parametrize('hidden,inner', [(256, 320), (50, 30)])
def test_assignments_of_every_kind(hidden, inner):
    """An expert twice, none at all, all tokens to one, weights of zero and below, padding, and experts that are not there."""
    gen = generator(13, hidden)
    x, w = normal(gen, 12, hidden, dtype=F16), layer(gen, 5, hidden, inner)
    r = normal(gen, 12, hidden, dtype=F16)
    same = torch.full((12, 3), 4, dtype=torch.int32, device='cuda')
    weights = normal(gen, 12, 3)
    check_layer(x, same, weights, *w)
    some = same.clone()
    some[:, 1], some[3], some[5, 0], some[11] = 2, -1, -7, -1
    weights[4] = 0
    got = check_layer(x, some, weights, *w, residual=r)
    assert torch.equal(got[3], r[3]) and torch.equal(got[11], r[11])
    assert not check_layer(x, torch.full_like(same, -1), weights, *w).any()
    assert ffi.func('b200q_check_status')() == ffi.OK
    beyond = some.clone()
    beyond[5, 0], beyond[7, 2] = 5, 2 ** 31 - 1
    passed = some.clone()
    passed[7, 2] = -1
    assert torch.equal(hidet_b200.mixture_of_experts(x, beyond, weights, *w), hidet_b200.mixture_of_experts(x, passed, weights, *w))
    with pytest.raises(ffi.BackendException, match='expert'):
        ffi.func('b200q_check_status')()
    none = hidet_b200.mixture_of_experts(x, some[:, :0], weights[:, :0], *w, residual=r)
    assert torch.equal(none, r)
    assert hidet_b200.mixture_of_experts(x[:0], some[:0], weights[:0], *w).shape == (0, hidden)


@pytest.mark.parametrize('dtype', [F16, BF16])
def test_values_of_any_size(dtype):
    """Tokens of unlike size beside one another, and hidden values beyond float16's range."""
    gen = generator(14)
    x = normal(gen, 10, 512, dtype=F32)
    x *= torch.logspace(-4, 2 if dtype == F16 else 5, 10, device='cuda')[:, None]
    gate_up, s1, down, s2 = layer(gen, 4, 512, 384)
    s1 = (s1.float() * 20).to(F16)
    experts, weights = choices(gen, 10, 4, 2)
    x = x.to(dtype)
    s2 = s2.float() * 1e-6
    s1 = s1.float()
    got = hidet_b200.mixture_of_experts(x, experts, weights, gate_up, s1, down, s2)
    want, bound = ref.experts(x, experts, weights, gate_up, s1, down, s2, None)
    ref.check(got, want, bound)
    h = (x.double() @ (gate_up[0].double() * s1[0].double()[:, None]).t()).abs().max()
    assert h > 1e3


@pytest.mark.parametrize('tokens', [8, 80])
def test_small_tokens_with_small_scales(tokens):
    """Sums whose power of two and scale are small together, below float's range, but not what they stand for."""
    gen = generator(24)
    x = (normal(gen, tokens, 512) * torch.logspace(-15, -12, tokens, device='cuda')[:, None]).to(BF16)
    w = layer(gen, 4, 512, 384)
    check_layer(x, *choices(gen, tokens, 4, 2), w[0], w[1].float() * 20, w[2], w[3].float() * 1e-6)


def test_tokens_that_are_no_numbers_stay_among_themselves():
    gen = generator(15)
    x, w = normal(gen, 9, 256, dtype=BF16), layer(gen, 3, 256, 128)
    experts, weights = choices(gen, 9, 3, 2)
    clean = hidet_b200.mixture_of_experts(x, experts, weights, *w)
    x[4, 7], weights[6, 1] = float('nan'), float('nan')
    got = hidet_b200.mixture_of_experts(x, experts, weights, *w)
    assert got[4].isnan().all() and got[6].isnan().all()
    keep = [0, 1, 2, 3, 5, 7, 8]
    assert torch.equal(got[keep], clean[keep])


def test_layer_of_strided_operands():
    gen = generator(16)
    big, w = normal(gen, 4, 3, 300, dtype=F16), layer(gen, 3, 256, 128)
    experts, weights = choices(gen, 12, 3, 2)
    experts, weights = experts.view(4, 3, 2), weights.view(4, 3, 2)
    for x in (big[..., :256], big[..., 1:257], big[..., 5:261], big[:, :1, :256].expand(4, 3, 256)):
        want = hidet_b200.mixture_of_experts(x.contiguous(), experts, weights, *w, residual=x.contiguous())
        assert torch.equal(hidet_b200.mixture_of_experts(x, experts, weights, *w, residual=x), want)
    out = big[..., :256].contiguous()
    want = hidet_b200.mixture_of_experts(big[..., :256], experts, weights, *w, residual=out)
    assert torch.equal(hidet_b200.mixture_of_experts(big[..., :256], experts, weights, *w, residual=out, out=out), want) and torch.equal(out, want)
    place = big[..., :256].contiguous()  # a layer in its input's place
    assert torch.equal(hidet_b200.mixture_of_experts(place, experts, weights, *w, residual=place, out=place), hidet_b200.mixture_of_experts(big[..., :256], experts, weights, *w, residual=big[..., :256]))
    moved = torch.empty(w[0].numel() + 1, dtype=torch.int8, device='cuda')[1:].view(w[0].shape).copy_(w[0])  # a base that is not aligned
    got = hidet_b200.mixture_of_experts(big[..., :256], experts, weights, moved, *w[1:])
    ref.check(got.view(12, 256), *ref.experts(big[..., :256].reshape(12, 256), experts.view(12, 2), weights.view(12, 2), *w, None))


@pytest.mark.parametrize('tokens', [6, 300])
def test_layer_captured_on_other_streams_and_beside_itself(tokens):
    gen = generator(17)
    x, router, w = normal(gen, tokens, 512, dtype=F16), normal(gen, 16, 512, dtype=F16, std=0.05), layer(gen, 16, 512, 256)

    def step():
        experts, weights = hidet_b200.route_tokens(x, router, 4)
        return hidet_b200.mixture_of_experts(x, experts, weights, *w, residual=x)

    want = step()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graphs = [hidet_b200.CudaGraph(lambda: [x], lambda inputs: [step()]) for _ in range(2)]
    other = normal(gen, tokens, 512, dtype=F16)
    for values in (other, x.clone()):
        x.copy_(values)
        want = step()
        for graph in graphs:
            outs = graph.run_async([x])
            assert torch.equal(outs[0], want)
    assert ffi.func('b200q_check_status')() == ffi.OK


def test_refusals():
    gen = generator(18)
    x, router, w = normal(gen, 2, 32, dtype=F16), normal(gen, 4, 32, dtype=F16), layer(gen, 4, 32, 48)
    e, p = choices(gen, 2, 4, 2)
    r, f = hidet_b200.route_tokens, hidet_b200.mixture_of_experts
    for call, text in ((lambda: r(x.int(), router, 2), 'float16'), (lambda: r(x, router[:, :31], 2), 'router'), (lambda: r(x, router.to(BF16), 2), 'router'), (lambda: r(x, router, 0), 'top_k'),
                       (lambda: r(x, router, 5), 'top_k'), (lambda: r(x, router, True), 'top_k'), (lambda: r(x, router, 2 ** 70), 'top_k'), (lambda: r(x, router, -1), 'top_k'), (lambda: r(x, torch.zeros(1025, 32, dtype=F16, device='cuda'), 2), '1024'),
                       (lambda: f(x.float(), e, p, *w), 'float16'), (lambda: f(x, e.long(), p, *w), 'experts'), (lambda: f(x, e[:1], p, *w), 'experts'), (lambda: f(x, e, p.half(), *w), 'weights'),
                       (lambda: f(x, e, p[:, :1], *w), 'weights'), (lambda: f(x, e, p, w[0][:, 1:], *w[1:]), 'gate_up'), (lambda: f(x, e, p, w[0], w[1], w[2][:, :, :47], w[3]), 'down'),
                       (lambda: f(x, e, p, w[0], w[1].float(), *w[2:]), 'scales'), (lambda: f(x, e, p, w[0], w[1][:, :95], *w[2:]), 'scales'), (lambda: f(x, e, p, *w, residual=x.float()), 'residual'),
                       (lambda: f(x, e, p, *w, out=x.float()), 'out')):
        with pytest.raises(ValueError, match=text):
            call()


def test_tokens_far_apart_and_weights_beyond_32_bits():
    gen = generator(19)
    x, router = far_rows(gen, 3, 512, (1 << 30) + 8, BF16), normal(gen, 24, 512, dtype=BF16)
    got, want = hidet_b200.route_tokens(x, router, 4), hidet_b200.route_tokens(x.contiguous(), router, 4)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    w = layer(gen, 24, 512, 272)
    assert torch.equal(hidet_b200.mixture_of_experts(x, *got, *w, residual=x), hidet_b200.mixture_of_experts(x.contiguous(), *got, *w, residual=x.contiguous()))
    del x
    count, hidden, inner = 40, 8192, 7008  # 4.6 and 2.3 GB
    last = layer(gen, 1, hidden, inner)
    gate_up, down = torch.empty(count, 2 * inner, hidden, dtype=torch.int8, device='cuda'), torch.empty(count, hidden, inner, dtype=torch.int8, device='cuda')
    gate_up[-1:], down[-1:] = last[0], last[2]
    x, weights = normal(gen, 2, hidden, dtype=F16), torch.ones(2, 1, device='cuda')
    chosen = torch.full((2, 1), count - 1, dtype=torch.int32, device='cuda')
    got = hidet_b200.mixture_of_experts(x, chosen, weights, gate_up, last[1].expand(count, -1), down, last[3].expand(count, -1))
    assert torch.equal(got, hidet_b200.mixture_of_experts(x, torch.zeros_like(chosen), weights, *last))


@pytest.mark.parametrize('hidden,inner', [(512, 256), (100, 36)])
def test_two_layers_at_once(hidden, inner):
    """Two streams with layers of their own, a hundred calls under way, beside linears on int8 tokens."""
    gen = generator(20, hidden)
    layers = [layer(gen, 8, hidden, inner) for _ in range(2)]
    xs = [normal(gen, n, hidden, dtype=F16) for n in (3, 40)]
    picks = [choices(gen, n, 8, 2) for n in (3, 40)]
    wq, scale = codes_of(gen, hidden, hidden), torch.full((hidden,), 1e-3, device='cuda')

    def step(i):
        y = hidet_b200.mixture_of_experts(xs[i], *picks[i], *layers[i])
        return hidet_b200.symmetric_quant_matmul_i8(*hidet_b200.quantize_tokens(y), wq, scale)

    want = [step(0), step(1)]
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(50):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])
    assert ffi.func('b200q_check_status')() == ffi.OK


def test_many_tokens_in_place_and_of_every_kind():
    """Results in the tokens' place, tokens that are no numbers, of any size and of large hidden values, assignments to nobody, beyond the layer and many times to one expert."""
    gen = generator(21)
    x, w = normal(gen, 300, 512, dtype=BF16), layer(gen, 6, 512, 272)
    experts, weights = choices(gen, 300, 6, 2)
    clean = check_layer(x, experts, weights, *w, residual=x)
    place = x.clone()
    assert torch.equal(hidet_b200.mixture_of_experts(place, experts, weights, *w, residual=place, out=place), clean) and torch.equal(place, clean)
    odd = x.clone()
    odd[4, 7], odd[100], odd[299, 0] = float('nan'), float('inf'), float('-inf')
    broken = weights.clone()
    broken[6, 1] = float('nan')
    got = hidet_b200.mixture_of_experts(odd, experts, broken, *w, residual=x)
    bad = torch.zeros(300, dtype=torch.bool, device='cuda')
    bad[[4, 6, 100, 299]] = True
    assert got[bad].isnan().all() and torch.equal(got[~bad], clean[~bad])
    sizes = (x.float() * torch.logspace(-30, 3, 300, device='cuda')[:, None]).to(BF16)
    sizes[17] = 0
    check_layer(sizes, experts, weights, w[0], w[1].float() * 20, w[2], w[3].float() * 1e-6)
    nobody = torch.full_like(experts, -1)
    assert torch.equal(hidet_b200.mixture_of_experts(x, nobody, weights, *w, residual=x), x) and not hidet_b200.mixture_of_experts(x, nobody, weights, *w).any()
    assert ffi.func('b200q_check_status')() == ffi.OK
    beyond, passed = experts.clone(), experts.clone()
    beyond[8, 0], beyond[200, 1], passed[8, 0], passed[200, 1] = 6, 2 ** 31 - 1, -1, -2
    assert torch.equal(hidet_b200.mixture_of_experts(x, beyond, weights, *w), hidet_b200.mixture_of_experts(x, passed, weights, *w))
    with pytest.raises(ffi.BackendException, match='expert'):
        ffi.func('b200q_check_status')()


@pytest.mark.parametrize('tokens,top', [(1, 1500), (3, 700), (2, 4096), (70, 150)])
def test_tokens_of_many_assignments(tokens, top):
    gen = generator(22, tokens, top)
    x, w = normal(gen, tokens, 128, dtype=F16), layer(gen, 5, 128, 64)
    experts = torch.randint(-1, 5, (tokens, top), generator=gen, device='cuda', dtype=torch.int32)
    check_layer(x, experts, torch.rand((tokens, top), generator=gen, device='cuda') / top, *w)


def test_layers_share_a_workspace_in_turn():
    """Few tokens, many and unaligned ones, and linears, in every order on one stream."""
    gen = generator(23)
    calls = []
    for tokens, count, top, hidden, inner in ((2, 8, 2, 512, 768), (200, 8, 2, 512, 768), (64, 4, 4, 256, 512), (5, 3, 2, 50, 30), (1000, 16, 4, 128, 64)):
        x, w, picks = normal(gen, tokens, hidden, dtype=F16), layer(gen, count, hidden, inner), choices(gen, tokens, count, top)
        calls.append(lambda x=x, w=w, picks=picks: hidet_b200.mixture_of_experts(x, *picks, *w))
    for m in (3, 40):
        a, wq, scale = normal(gen, m, 4096, dtype=F16), codes_of(gen, 4096, 512), torch.full((512,), 1e-3, dtype=F16, device='cuda')
        calls.append(lambda a=a, wq=wq, scale=scale: hidet_b200.symmetric_quant_matmul(a, wq, scale))
    want = [call() for call in calls]
    for i in torch.randint(0, len(calls), (200,), generator=torch.Generator().manual_seed(3)).tolist():
        assert torch.equal(calls[i](), want[i])
    assert ffi.func('b200q_check_status')() == ffi.OK
