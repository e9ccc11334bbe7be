"""Linears on int8 tokens and layers of experts, as programs that use this package run them.

listed() names a fixed set of cases, draw() gives further ones of the same ranges, prepare() makes what a program holds
before the call, run() is one pass: in plain torch operations, or through the package's entry points where `own` is true.
exact() computes the same from the definitions in 64 bits, work() counts the bytes and operations a pass cannot do without.

Kinds of case:
    project  quantize_tokens of a layer's input (behind an RMS norm, or as it is), then symmetric_quant_matmul_i8 with an int8
             weight, and what follows it: a bias, the gate / up pairing, a residual
    experts  route_tokens, then mixture_of_experts, of the tokens of a decode step

code = rint(y * (127 / amax)), value = code * (amax / 127), amax over a token's elements of y; a weight has one scale for each
output channel.  With the pairing the weight's channels are (gate_j, up_j) pairs and the result silu(gate) * up.
"""
import math

import torch

own = False

DTYPES = {'float16': torch.float16, 'bfloat16': torch.bfloat16, 'float32': torch.float32}
EPS = 1e-5


def listed():
    return [
        # The output projection of the batch-1 decoder: launch and host time.
        dict(name='project_1x4096x4096', kind='project', tokens=1, inner=4096, outer=4096, layout='KN', norm=False, bias=False, pairs=False, residual=True,
             dtype='float16'),
        # Gate and up of a batch of sequences, one token each, behind the norm.
        dict(name='project_16x4096x22016_norm_pairs', kind='project', tokens=16, inner=4096, outer=22016, layout='KN', norm=True, bias=False, pairs=True,
             residual=False, dtype='float16'),
        # A short prompt of an odd length, weights as torch's linear layers keep them, with a bias.
        dict(name='project_333x4096x12288_bias', kind='project', tokens=333, inner=4096, outer=12288, layout='NK', norm=True, bias=True, pairs=False,
             residual=False, dtype='bfloat16'),
        # The feed-forward part over a 2048-token prompt, both of its linears.
        dict(name='project_2048x4096x22016_norm_pairs', kind='project', tokens=2048, inner=4096, outer=22016, layout='KN', norm=True, bias=False, pairs=True,
             residual=False, dtype='float16'),
        dict(name='project_2048x11008x4096', kind='project', tokens=2048, inner=11008, outer=4096, layout='KN', norm=False, bias=False, pairs=False,
             residual=True, dtype='float16'),
        # A long prompt at a 70B-class layer's width.
        dict(name='project_8192x8192x10240_nk', kind='project', tokens=8192, inner=8192, outer=10240, layout='NK', norm=True, bias=False, pairs=False,
             residual=False, dtype='bfloat16'),
        # One token, a few large experts.
        dict(name='experts_1_of_8x4096x14336', kind='experts', tokens=1, experts=8, top=2, hidden=4096, inner=14336, dtype='float16'),
        # A few tokens, many small experts.
        dict(name='experts_7_of_64x2048x1408', kind='experts', tokens=7, experts=64, top=6, hidden=2048, inner=1408, dtype='bfloat16'),
        # A serving batch: most experts have a token.
        dict(name='experts_48_of_128x2048x768', kind='experts', tokens=48, experts=128, top=8, hidden=2048, inner=768, dtype='bfloat16'),
        # A serving batch over large experts, several tokens each.
        dict(name='experts_32_of_8x4096x14336', kind='experts', tokens=32, experts=8, top=2, hidden=4096, inner=14336, dtype='float16'),
    ]


MOST_PRODUCTS = 8192 * 8192 * 10240
MOST_WEIGHTS = 3 * 8 * 4096 * 14336


def _log(rng, low, high, step=1):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high))) / step)) * step


def draw(rng):
    kind = rng.choice(['project', 'project', 'experts'])
    dtype = rng.choice(['float16', 'bfloat16'])
    while True:
        if kind == 'project':
            pairs = rng.random() < 0.3
            c = dict(kind=kind, tokens=_log(rng, 1, 8192), inner=_log(rng, 256, 16384, 16), outer=_log(rng, 256, 28672, 16), layout=rng.choice(['KN', 'NK']),
                     norm=rng.random() < 0.5, bias=rng.random() < 0.3, pairs=pairs, residual=not pairs and rng.random() < 0.4, dtype=dtype)
            if c['tokens'] * c['inner'] * c['outer'] <= MOST_PRODUCTS and c['inner'] * c['outer'] <= 1 << 28:
                return c
        else:
            experts = rng.choice([4, 8, 16, 32, 64, 128])
            c = dict(kind=kind, tokens=_log(rng, 1, 64), experts=experts, top=min(experts, rng.choice([1, 2, 2, 4, 6, 8])), hidden=_log(rng, 512, 8192, 16),
                     inner=_log(rng, 256, 14336, 16), dtype=dtype)
            if 3 * experts * c['hidden'] * c['inner'] <= MOST_WEIGHTS:
                return c


def work(case):
    size = DTYPES[case['dtype']].itemsize
    tokens = case['tokens']
    if case['kind'] == 'project':
        k, n = case['inner'], case['outer']
        out = n // 2 if case['pairs'] else n
        bytes_ = size * tokens * k + k * n + 2 * n + size * tokens * out * (2 if case['residual'] else 1) + (size * k if case['norm'] else 0) + (size * n if case['bias'] else 0)
        return {'bytes': bytes_, 'flops': 2.0 * tokens * k * n}
    experts, top, hidden, inner = case['experts'], case['top'], case['hidden'], case['inner']
    chosen = experts * (1.0 - (1.0 - top / experts) ** tokens)  # experts that have a token, as routing spreads them
    bytes_ = chosen * (3 * hidden * inner + 2 * (2 * inner + hidden)) + size * hidden * (2 * tokens + experts) + 8 * tokens * top
    return {'bytes': int(bytes_), 'flops': 2.0 * tokens * hidden * (3 * inner * top + experts)}


# ---- prepare ----

def _normal(gen, shape, std, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device='cuda', dtype=torch.float32).mul_(std).to(dtype)


def _weight(gen, outer, inner):
    """int8 [outer, inner] and float16 [outer]: normal weights of 0.02, some channels larger than others."""
    codes = torch.empty((outer, inner), dtype=torch.int8, device='cuda')
    scales = torch.empty(outer, dtype=torch.float16, device='cuda')
    for at in range(0, outer, 16384):
        rows = slice(at, min(at + 16384, outer))
        w = _normal(gen, codes[rows].shape, 0.02) * _normal(gen, scales[rows].shape, 0.2).exp()[:, None]
        scales[rows] = w.abs().amax(1) / 127
        codes[rows] = (w / scales[rows].float()[:, None]).round().clamp(-127, 127).to(torch.int8)
    return codes, scales


def _hidden(gen, tokens, width, dtype):
    """Rows of a residual stream: channels of unlike size, a few of them far larger."""
    gain = _normal(gen, (width,), 0.4).exp()
    gain[torch.randint(0, width, (max(1, width // 512),), generator=gen, device='cuda')] *= 8
    return (_normal(gen, (tokens, width), 1.0) * gain).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    dtype, tokens = DTYPES[case['dtype']], case['tokens']
    if case['kind'] == 'project':
        weight, scale = _weight(gen, case['outer'], case['inner'])
        if case['layout'] == 'KN':
            weight = weight.t().contiguous()
        out = case['outer'] // 2 if case['pairs'] else case['outer']
        return {'kind': 'project', 'x': _hidden(gen, tokens, case['inner'], dtype), 'weight': weight, 'scale': scale, 'layout': case['layout'], 'pairs': case['pairs'],
                'norm': (1 + _normal(gen, (case['inner'],), 0.1)).to(dtype) if case['norm'] else None,
                'bias': _normal(gen, (case['outer'],), 0.1, dtype) if case['bias'] else None,
                'residual': _normal(gen, (tokens, out), 1.0, dtype) if case['residual'] else None}
    experts, hidden, inner, top = case['experts'], case['hidden'], case['inner'], case['top']
    gate_up, down = _weight(gen, experts * 2 * inner, hidden), _weight(gen, experts * hidden, inner)
    x = _normal(gen, (tokens, hidden), 1.0, dtype)
    router = _normal(gen, (experts, hidden), 1.5 * hidden ** -0.5, dtype)
    # a token that stands between two choices takes its values from one that does not
    if top < experts:
        order = (x.double() @ router.double().t()).sort(-1, descending=True)[0]
        close = (order[:, :top] - order[:, 1:top + 1]).amin(-1) < 1e-4
        x = torch.where(close[:, None], x[(~close).int().argmax()], x)
    return {'kind': 'experts', 'x': x, 'router': router, 'top': top, 'gate_up': gate_up[0].view(experts, 2 * inner, hidden), 'gate_up_scale': gate_up[1].view(experts, 2 * inner),
            'down': down[0].view(experts, hidden, inner), 'down_scale': down[1].view(experts, hidden)}


# ---- run ----

def _plain_project(s):
    y = s['x'].float()
    if s['norm'] is not None:
        y = y * ((y * y).mean(-1, keepdim=True) + EPS).rsqrt() * s['norm'].float()
    amax = y.abs().amax(-1, keepdim=True)
    codes = torch.round(y * (127.0 / amax))
    weight = s['weight'].float()
    c = codes @ (weight if s['layout'] == 'KN' else weight.t())
    c = c * (amax / 127.0) * s['scale'].float()
    if s['bias'] is not None:
        c = c + s['bias'].float()
    if s['pairs']:
        gate, up = c[:, 0::2], c[:, 1::2]
        c = gate / (1 + torch.exp(-gate)) * up
    if s['residual'] is not None:
        c = c + s['residual'].float()
    return c.to(s['x'].dtype)


def _plain_experts(s):
    x, top = s['x'].float(), s['top']
    logits = x @ s['router'].float().t()
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    chosen = torch.sort(logits, dim=-1, descending=True, stable=True)[1][:, :top]
    weights = p.gather(1, chosen)
    weights = weights / weights.sum(-1, keepdim=True)
    out = torch.zeros_like(x)
    for e in range(s['router'].shape[0]):
        share = torch.where(chosen == e, weights, 0.0).sum(-1, keepdim=True)
        y = x @ s['gate_up'][e].float().t() * s['gate_up_scale'][e].float()
        gate, up = y[:, 0::2], y[:, 1::2]
        h = gate / (1 + torch.exp(-gate)) * up
        out += share * (h @ s['down'][e].float().t() * s['down_scale'][e].float())
    return out.to(s['x'].dtype), chosen.int(), weights


def run(state):
    s = state
    if not own:
        return _plain_project(s) if s['kind'] == 'project' else _plain_experts(s)
    import hidet_b200

    if s['kind'] == 'project':
        codes, scales = hidet_b200.quantize_tokens(s['x'], norm=s['norm'], eps=EPS)
        return hidet_b200.symmetric_quant_matmul_i8(codes, scales, s['weight'], s['scale'], weight_layout=s['layout'], bias=s['bias'], residual=s['residual'],
                                                    activation='silu_mul' if s['pairs'] else None, dtype=s['x'].dtype)
    experts, weights = hidet_b200.route_tokens(s['x'], s['router'], s['top'])
    out = hidet_b200.mixture_of_experts(s['x'], experts, weights, s['gate_up'], s['gate_up_scale'], s['down'], s['down_scale'])
    return out, experts, weights


# ---- exact ----

def _exact_project(s):
    x = s['x'].double()
    if s['norm'] is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * s['norm'].double()
    step = x.abs().amax(-1, keepdim=True) / 127
    codes = torch.where(step > 0, (x / step).round(), 0.0)
    scale = s['scale'].double()
    n = scale.shape[0]
    out = torch.empty((x.shape[0], n), dtype=torch.float64, device='cuda')
    for at in range(0, n, 4096):
        part = slice(at, min(at + 4096, n))
        w = s['weight'][:, part].double() if s['layout'] == 'KN' else s['weight'][part].double().t()
        out[:, part] = codes @ (w * scale[part]) * step
    if s['bias'] is not None:
        out += s['bias'].double()
    if s['pairs']:
        out = out.view(x.shape[0], n // 2, 2)
        out = out[..., 0] * torch.sigmoid(out[..., 0]) * out[..., 1]
    if s['residual'] is not None:
        out = out + s['residual'].double()
    return out


def _exact_experts(s):
    x = s['x'].double()
    p = torch.softmax(x @ s['router'].double().t(), -1)
    weights, chosen = p.topk(s['top'], -1)
    weights = weights / weights.sum(-1, keepdim=True)
    out = torch.zeros_like(x)
    for e in chosen.unique().tolist():
        token, place = (chosen == e).nonzero(as_tuple=True)
        y = (x[token] @ s['gate_up'][e].double().t()).mul(s['gate_up_scale'][e].double()).unflatten(-1, (-1, 2))
        h = y[..., 0] * torch.sigmoid(y[..., 0]) * y[..., 1]
        out.index_add_(0, token, weights[token, place][:, None] * (h @ s['down'][e].double().t()) * s['down_scale'][e].double())
    return out, chosen.int(), weights


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_project(state) if case['kind'] == 'project' else _exact_experts(state)
