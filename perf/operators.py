"""The operators of a decoder's verification step, as programs that use this package run them: rotary positions, the
quantized key/value cache (written, read back, attended to by a token or by a tree of drafted tokens) and the log
probabilities of given tokens.

listed() names a fixed set of cases, draw() gives further ones of the same ranges, prepare() makes what a program holds
before the call, run() is one pass: in plain torch operations, or through the package's entry points where `own` is true.
exact() computes the same from the definitions in 64 bits, work() counts the bytes and operations a pass cannot do without.

Kinds of case:
    rotary     rotary_embedding of the queries and keys of a fused projection's rows
    append     quantized_cache_append of those rows (queries and keys rotated on the way), then quantized_cache_read of them
    read       quantized_cache_read of a long prefix
    attention  quantized_cache_attention of one token a sequence, or of a tree of drafted tokens
    log_probs  token_log_probs: given tokens, the entropy of every row and its top alternatives

The cache is uint8 [pages, kv_heads, page_size / 16, 32 D + 128], a record for every 16 positions of a head: the codes of 16
rows of K and of 16 rows of V (a byte is code + 128), then their 16 + 16 float32 scales.  Inside row r the 16-byte chunks
stand in the order c ^ s(r): s(r) is the upper log2(gcd(D / 16, 8)) bits of the three bits (r3, r2, r0) of r for K and
(r2, r1, r0) for V.  code = rint(x * (127 / amax)), value = code * (amax / 127), amax over the D elements of a row.
"""
import math

import torch

own = False

DTYPES = {'float16': torch.float16, 'bfloat16': torch.bfloat16, 'float32': torch.float32}


def listed():
    return [
        # One token of the batch-1 decoder: launch and host time.  32 heads of 128, interleaved pairs.
        dict(name='rotary_1x32x128', kind='rotary', tokens=1, heads=32, kv_heads=32, dim=128, rotary_dim=128, layout='interleaved',
             scaling='none', dtype='float16'),
        # A 2048-token prompt at a 70B-class layer's heads, with positions scaled for a context four times as long.
        dict(name='rotary_2048x64x128_yarn', kind='rotary', tokens=2048, heads=64, kv_heads=8, dim=128, rotary_dim=128, layout='half',
             scaling='yarn', dtype='bfloat16'),
        # One decode step's token into the cache.
        dict(name='append_1x32x128', kind='append', tokens=1, heads=32, kv_heads=32, dim=128, rotary_dim=128, layout='interleaved',
             scaling='none', dtype='float16', page_size=64),
        # An odd number of tokens of several sequences, half of a small head rotated, small pages.
        dict(name='append_333x16x64_half', kind='append', tokens=333, heads=16, kv_heads=4, dim=64, rotary_dim=32, layout='half',
             scaling='linear', dtype='float16', page_size=16),
        # A long prompt.
        dict(name='append_8192x32x128', kind='append', tokens=8192, heads=32, kv_heads=8, dim=128, rotary_dim=128, layout='half',
             scaling='none', dtype='bfloat16', page_size=64),
        # A cached prefix back in 16 bits, for a dense pass over it.
        dict(name='read_16384x8x128', kind='read', tokens=16384, kv_heads=8, dim=128, dtype='float16', page_size=64),
        # Batch-1 decoding in the middle of the decoder configuration's 640 positions.
        dict(name='decode_1x32_at_577', kind='attention', batch=1, tokens=1, even=True, heads=32, kv_heads=32, dim=128, shortest=577,
             longest=577, dtype='float16', page_size=64, tree=False),
        # A serving batch with ragged contexts.
        dict(name='decode_32x64_to_8000', kind='attention', batch=32, tokens=1, even=True, heads=64, kv_heads=8, dim=128, shortest=90,
             longest=8000, dtype='bfloat16', page_size=64, tree=False),
        # One long document.
        dict(name='decode_1x64_at_131071', kind='attention', batch=1, tokens=1, even=True, heads=64, kv_heads=8, dim=128, shortest=131071,
             longest=131071, dtype='float16', page_size=128, tree=False),
        # Trees of up to 64 drafted tokens verified for eight sequences.
        dict(name='tree_8x64x32_to_4096', kind='attention', batch=8, tokens=64, even=False, heads=32, kv_heads=8, dim=128, shortest=500,
             longest=4096, dtype='float16', page_size=16, tree=True),
        # The token just sampled, with five alternatives.
        dict(name='log_probs_1x32000', kind='log_probs', rows=1, vocab=32000, given=1, top=5, dtype='float16'),
        # Scoring a long text, a vocabulary with two added tokens.
        dict(name='log_probs_2047x32002', kind='log_probs', rows=2047, vocab=32002, given=1, top=20, dtype='bfloat16'),
    ]


MOST_ROTARY = 2048 * 72 * 128
MOST_APPEND = 8192 * 48 * 128
MOST_READ = 16384 * 8 * 128
MOST_ATTENTION = 131071 * 8 * 128   # key and value elements read
MOST_SCORES = 8 * 64 * 32 * 2300    # (query row, key) pairs
MOST_LOGITS = 2047 * 32002


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(['rotary', 'append', 'append', 'read', 'attention', 'attention', 'attention', 'attention', 'log_probs', 'log_probs'])
    dtype = rng.choice(['float16', 'bfloat16'])
    if kind == 'log_probs':
        while True:
            c = dict(kind=kind, rows=_log(rng, 1, 3000), vocab=_log(rng, 500, 160000), given=rng.choice([1, 1, 1, 4]), top=rng.choice([0, 1, 5, 20, 32]),
                     dtype=rng.choice(['float16', 'bfloat16', 'float32']))
            if c['rows'] * c['vocab'] <= (MOST_LOGITS if c['dtype'] != 'float32' else MOST_LOGITS // 2):
                return c
    kv_heads, group, dim = rng.choice([1, 2, 4, 8, 8, 16, 32]), rng.choice([1, 2, 4, 4, 5, 8]), rng.choice([64, 128, 128, 128])
    page_size = rng.choice([16, 32, 64, 64, 128, 256])
    if kind == 'read':
        while True:
            c = dict(kind=kind, tokens=_log(rng, 1, 16384), kv_heads=kv_heads, dim=dim, dtype=dtype, page_size=page_size)
            if c['tokens'] * kv_heads * dim <= MOST_READ:
                return c
    if kind in ('rotary', 'append'):
        most = MOST_ROTARY if kind == 'rotary' else MOST_APPEND
        while True:
            c = dict(kind=kind, tokens=_log(rng, 1, 8192), heads=kv_heads * group, kv_heads=kv_heads, dim=dim, rotary_dim=rng.choice([dim, dim, dim // 2]),
                     layout=rng.choice(['half', 'interleaved']), scaling=rng.choice(['none', 'linear', 'ntk', 'yarn']), dtype=dtype)
            if kind == 'append':
                c['page_size'] = page_size
            if c['tokens'] * (group + (2 if kind == 'append' else 1)) * kv_heads * dim <= most:
                return c
    tree = rng.random() < 0.5
    while True:
        longest = _log(rng, 16, 131071)
        c = dict(kind=kind, batch=_log(rng, 1, 64), tokens=_log(rng, 2, 64) if tree else 1, even=not tree or rng.random() < 0.3, heads=kv_heads * group,
                 kv_heads=kv_heads, dim=dim, shortest=max(1, int(longest * rng.choice([0.05, 0.3, 1.0]))), longest=longest, dtype=dtype,
                 page_size=page_size, tree=tree)
        # the longest sequence counts for all: the plain form pads to it
        if c['batch'] * longest * kv_heads * dim <= MOST_ATTENTION and c['batch'] * c['tokens'] * c['heads'] * longest <= MOST_SCORES:
            return c


# ---- sizes that follow from a case ----

def _spread(low, high, n):
    """n lengths between low and high, the longest first and the others in no order."""
    step = next(s for s in (7, 11, 13, 17) if n % s) if n > 1 else 1
    return [high - (high - low) * ((step * i) % n) // max(1, n - 1) for i in range(n)]


def _tokens(case):
    """Drafted tokens of every sequence."""
    return [case['tokens']] * case['batch'] if case['even'] else _spread(max(1, case['tokens'] - case['tokens'] // 4), case['tokens'], case['batch'])


def _lengths(case):
    """Cached positions of every sequence, the drafted tokens among them."""
    return [max(n, t) for n, t in zip(_spread(case['shortest'], case['longest'], case['batch']), _tokens(case))]


def work(case):
    kind = case['kind']
    if kind == 'log_probs':
        rows, n = case['rows'], case['rows'] * case['vocab']
        out = rows * (4 + 4 * case['given'] + 12 * case['top'])
        return {'bytes': n * DTYPES[case['dtype']].itemsize + 8 * rows * case['given'] + out, 'flops': 6.0 * n}
    dim, kv_heads = case['dim'], case['kv_heads']
    record = 2 * dim + 8  # codes and scales of one position of one head
    if kind == 'read':
        return {'bytes': case['tokens'] * (kv_heads * (record + 4 * dim) + 8), 'flops': 2.0 * case['tokens'] * kv_heads * dim}
    heads = case['heads']
    if kind in ('rotary', 'append'):
        tokens, rotated = case['tokens'], heads + kv_heads
        table = 4 * tokens * case['rotary_dim']
        if kind == 'rotary':
            return {'bytes': tokens * (4 * rotated * dim + 8) + table, 'flops': 3.0 * tokens * rotated * case['rotary_dim']}
        # rows in, queries out, records written, then read again and given back in 16 bits
        bytes_ = tokens * (2 * (2 * heads + 2 * kv_heads) * dim + 16 + kv_heads * (2 * record + 4 * dim) + 8) + table
        return {'bytes': bytes_, 'flops': tokens * (3.0 * rotated * case['rotary_dim'] + 10.0 * kv_heads * dim)}
    lengths, tokens = _lengths(case), _tokens(case)
    rows = sum(tokens)
    pages = sum(-(-n // case['page_size']) for n in lengths)
    bytes_ = sum(lengths) * kv_heads * record + 4 * pages + 4 * rows * heads * dim + 4 * rows * heads + (sum(t * t for t in tokens) if case['tree'] else 0)
    return {'bytes': bytes_, 'flops': 4.0 * dim * heads * sum(t * n for t, n in zip(tokens, lengths))}


# ---- the cache's layout, in plain torch ----

def _order(dim, device):
    """Where the 16-byte chunks of the 16 rows of a record stand: [16, dim / 16] for K and for V (each its own inverse)."""
    r = torch.arange(16, device=device)
    low = 3 - int(math.log2(math.gcd(dim // 16, 8)))
    k = (((r >> 1) & 6) | (r & 1)) >> low
    v = (r & 7) >> low
    c = torch.arange(dim // 16, device=device)
    return c ^ k[:, None], c ^ v[:, None]


def _parts(cache, dim):
    """Views of a cache's codes [..., 16, dim / 16, 16] and scales [..., 16], of K and then of V."""
    k, v = (cache[..., i * 16 * dim:(i + 1) * 16 * dim].unflatten(-1, (16, dim // 16, 16)) for i in (0, 1))
    ks, vs = (cache[..., 32 * dim + i * 64:32 * dim + (i + 1) * 64].view(torch.float32) for i in (0, 1))
    return k, v, ks, vs


def _quantized(x):
    """Rows of x -> (bytes, scales), in x's own precision."""
    amax = x.abs().amax(-1, keepdim=True)
    limit = torch.full_like(amax, 127.0)
    code = torch.where(amax > 0, torch.round(x * (limit / amax)), torch.zeros_like(x))
    return code, (amax / limit)[..., 0]


def _rows_of(cache, slots, dim):
    """The restored rows [tokens, kv_heads, dim] of K and of V at slots, in float32."""
    page_size = cache.shape[2] * 16
    page, block, row = slots // page_size, slots % page_size // 16, slots % 16
    k, v, ks, vs = _parts(cache, dim)
    restored = []
    for codes, scales, order in zip((k, v), (ks, vs), _order(dim, cache.device)):
        rows = codes[page, :, block, row]                                            # [tokens, kv_heads, dim / 16, 16]
        rows = rows.gather(2, order[row][:, None, :, None].expand(rows.shape)).flatten(2)
        restored.append((rows.float() - 128.0) * scales[page, :, block, row][..., None])
    return restored


def _write(cache, slots, k, v, dim):
    page_size = cache.shape[2] * 16
    page, block, row = slots // page_size, slots % page_size // 16, slots % 16
    for x, codes, scales, order in zip((k, v), _parts(cache, dim)[:2], _parts(cache, dim)[2:], _order(dim, cache.device)):
        code, scale = _quantized(x)
        stored = (code + 128.0).to(torch.uint8).unflatten(-1, (dim // 16, 16))
        codes[page, :, block, row] = stored.gather(2, order[row][:, None, :, None].expand(stored.shape))
        scales[page, :, block, row] = scale


# ---- prepare ----

def _normal(gen, shape, std, dtype):
    return torch.randn(shape, generator=gen, device='cuda', dtype=torch.float32).mul_(std).to(dtype)


def _frequencies(dim, scaling, positions):
    """Angle per position of every pair, in 64 bits, and the factor of its cosine and sine: contexts four times as long."""
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    base, factor = 10000.0, 4.0
    if scaling == 'ntk':
        base = base * factor ** (dim / (dim - 2))
    f = base ** (-i / dim)
    if scaling == 'linear':
        f = f / factor
    if scaling != 'yarn':
        return f, 1.0
    original = positions / factor
    low, high = (dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0))
    low, high = max(math.floor(low), 0), min(math.ceil(high), dim - 1)
    ramp = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0


def _table(dim, scaling, positions=16384):
    """The cosines and then the sines of every position, as a program makes them once."""
    f, by = _frequencies(dim, scaling, positions)
    angle = torch.arange(positions, device='cuda', dtype=torch.float64)[:, None] * f.cuda()
    return torch.cat([angle.cos() * by, angle.sin() * by], -1).float()


def _empty_cache(slots, kv_heads, dim, page_size):
    return torch.zeros((-(-slots // page_size), kv_heads, page_size // 16, 32 * dim + 128), dtype=torch.uint8, device='cuda')


def _filled_cache(gen, slots, kv_heads, dim, page_size):
    """A cache whose every row is written, key channels of unlike size as projections give them."""
    cache = _empty_cache(slots, kv_heads, dim, page_size)
    gain = _normal(gen, (kv_heads, dim), 0.5, torch.float32).exp()
    parts = _parts(cache, dim)
    for i, order in enumerate(_order(dim, 'cuda')):
        for first in range(0, cache.shape[0], max(1, 65536 // page_size)):
            at = slice(first, first + max(1, 65536 // page_size))
            x = torch.randn(parts[i][at].flatten(-2).shape, generator=gen, device='cuda')
            code, scale = _quantized(x * gain[:, None, None] if i == 0 else x)
            stored = (code + 128.0).to(torch.uint8).unflatten(-1, (dim // 16, 16))
            parts[i][at] = stored.gather(-2, order[:, :, None].expand(stored.shape))
            parts[2 + i][at] = scale
    return cache


def _trees(gen, tokens):
    """A mask row for every drafted token: its ancestors and itself.  The first token of a sequence is the root."""
    n, width = len(tokens), max(tokens)
    pick = torch.rand((n, width), generator=gen, device='cuda').cpu()
    mask = torch.zeros((n, width, width), dtype=torch.bool)
    mask[:, 0, 0] = True
    each = torch.arange(n)
    for i in range(1, width):
        parent = (pick[:, i].sqrt() * i).long()  # late tokens more often than early ones
        mask[:, i] = mask[each, parent]
        mask[:, i, i] = True
    return torch.cat([mask[b, :t] for b, t in enumerate(tokens)]).cuda()


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    kind, dtype = case['kind'], DTYPES[case['dtype']]
    if kind == 'log_probs':
        logits = _normal(gen, (case['rows'], case['vocab']), 2.5, torch.float32)
        logits *= torch.rand((case['rows'], 1), generator=gen, device='cuda') + 0.5
        tokens = torch.randint(0, case['vocab'], (case['rows'], case['given']), generator=gen, device='cuda')
        likely = torch.rand((case['rows'], case['given']), generator=gen, device='cuda') < 0.7
        tokens = torch.where(likely, logits.argmax(-1, keepdim=True), tokens)
        return {'kind': kind, 'logits': logits.to(dtype), 'tokens': tokens, 'top': case['top']}
    kv_heads, dim = case['kv_heads'], case['dim']
    if kind == 'read':
        cache = _filled_cache(gen, case['tokens'] + 1000, kv_heads, dim, case['page_size'])
        pages = torch.randperm(cache.shape[0], generator=gen, device='cuda')
        slots = (pages[:, None] * case['page_size'] + torch.arange(case['page_size'], device='cuda')).flatten()[:case['tokens']].contiguous()
        return {'kind': kind, 'cache': cache, 'slots': slots, 'dim': dim, 'dtype': dtype}
    heads = case['heads']
    if kind in ('rotary', 'append'):
        tokens = case['tokens']
        qkv = _normal(gen, (tokens, (heads + 2 * kv_heads) * dim), 1.0, dtype)
        q, k, v = (x.unflatten(-1, (-1, dim)) for x in qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], -1))
        table = _table(case['rotary_dim'], case['scaling'])
        first = torch.randint(0, table.shape[0] - tokens, (1,), generator=gen, device='cuda')
        state = {'kind': kind, 'q': q, 'k': k, 'positions': first + torch.arange(tokens, device='cuda'), 'table': table, 'layout': case['layout']}
        if kind == 'rotary':
            return state
        cache = _empty_cache(tokens + 1000, kv_heads, dim, case['page_size'])
        pages = torch.randperm(cache.shape[0], generator=gen, device='cuda')
        slots = (pages[:, None] * case['page_size'] + torch.arange(case['page_size'], device='cuda')).flatten()[:tokens].contiguous()
        return dict(state, v=v, cache=cache, slots=slots, dim=dim, dtype=dtype)
    lengths, tokens, page_size = _lengths(case), _tokens(case), case['page_size']
    used = [-(-n // page_size) for n in lengths]
    cache = _filled_cache(gen, (sum(used) + 8) * page_size, kv_heads, dim, page_size)
    order = torch.randperm(cache.shape[0], generator=gen, device='cuda').to(torch.int32)
    table = torch.zeros((len(lengths), max(used)), dtype=torch.int32, device='cuda')
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [sum(tokens[:b]) for b in range(len(tokens) + 1)]
    return {'kind': kind, 'q': _normal(gen, (sum(tokens), heads, dim), 1.5, dtype), 'cache': cache, 'table': table, 'dim': dim,
            'lengths': torch.tensor(lengths, dtype=torch.int32, device='cuda'),
            'starts': torch.tensor(starts, dtype=torch.int32, device='cuda') if case['tree'] else None,
            'most': max(tokens), 'mask': _trees(gen, tokens) if case['tree'] else None}


# ---- run ----

def _rotated(x, positions, table, layout):
    """x [tokens, heads, dim] in float32, its first table.shape[1] elements rotated."""
    x, half = x.float(), table.shape[1] // 2
    cos, sin = table[positions][:, None, :half], table[positions][:, None, half:]
    a, b = (x[..., :half], x[..., half:2 * half]) if layout == 'half' else (x[..., 0:2 * half:2], x[..., 1:2 * half:2])
    a, b = a * cos - b * sin, b * cos + a * sin
    return torch.cat([torch.cat([a, b], -1) if layout == 'half' else torch.stack([a, b], -1).flatten(-2), x[..., 2 * half:]], -1)


def _plain_attention(state):
    q, cache, table, lengths, dim, most = (state[n] for n in ('q', 'cache', 'table', 'lengths', 'dim', 'most'))
    k, v, ks, vs = _parts(cache[table.long()], dim)             # [batch, pages, kv_heads, blocks, 16, ...]

    def restored(codes, scales, order):
        rows = codes.gather(-2, order[:, :, None].expand(codes.shape)).flatten(-2).float().sub_(128.0).mul_(scales[..., None])
        return rows.transpose(1, 2).flatten(2, 4)               # [batch, kv_heads, positions, dim]

    k_order, v_order = _order(dim, q.device)
    k, v = restored(k, ks, k_order), restored(v, vs, v_order)
    batch, kv_heads, positions, _ = k.shape
    group = q.shape[1] // kv_heads
    starts = state['starts'].long() if state['starts'] is not None else torch.arange(batch + 1, device=q.device)
    each = torch.arange(most, device=q.device)
    there = each < (starts[1:] - starts[:-1])[:, None]          # [batch, most]: this token is one of the sequence's
    rows = (starts[:-1, None] + each).clamp(max=q.shape[0] - 1)
    queries = q.float()[rows].unflatten(2, (kv_heads, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    scores = (queries @ k.transpose(-1, -2)).mul_(dim ** -0.5).unflatten(2, (most, group))  # [batch, kv_heads, most, group, positions]
    at = torch.arange(positions, device=q.device)
    old = lengths.long() - (starts[1:] - starts[:-1])           # positions in front of the drafted ones
    seen = (at < lengths[:, None])[:, None, :].expand(batch, most, positions)
    if state['mask'] is not None:
        drafted = at - old[:, None]                             # [batch, positions]
        allowed = state['mask'][rows].gather(2, drafted.clamp(0, state['mask'].shape[1] - 1)[:, None, :].expand(batch, most, positions))
        seen = seen & ((drafted < 0)[:, None, :] | allowed)
    scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = ((p.flatten(2, 3) @ v).unflatten(2, (most, group)) / total).permute(0, 2, 1, 3, 4).flatten(2, 3)
    lse = (total.log() + top)[..., 0].permute(0, 2, 1, 3).flatten(2)
    return out[there].to(q.dtype), lse[there]


def _plain_log_probs(logits, tokens, top):
    x = logits.float()
    most = x.amax(-1, keepdim=True)
    p = (x - most).exp()
    total = p.sum(-1, keepdim=True)
    lse = most + total.log()
    entropy = total.log()[:, 0] - ((x - most) * p).sum(-1) / total[:, 0]
    # values in their order, equal ones by index: one whole number for both
    bits = x.view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() * (1 << 32) + (0xffffffff - torch.arange(x.shape[1], device=x.device))
    index = 0xffffffff - (key.topk(top, -1)[0] & 0xffffffff)
    return x.gather(1, tokens) - lse, entropy, x.gather(1, index) - lse, index


def run(state):
    kind = state['kind']
    if own:
        import hidet_b200

        if kind == 'rotary':
            return hidet_b200.rotary_embedding(state['q'], state['k'], state['positions'], state['table'], layout=state['layout'])
        if kind == 'append':
            q = hidet_b200.quantized_cache_append(state['cache'], state['k'], state['v'], state['slots'], q=state['q'], positions=state['positions'],
                                                  table=state['table'], layout=state['layout'])
            return (q,) + hidet_b200.quantized_cache_read(state['cache'], state['slots'], state['dtype'])
        if kind == 'read':
            return hidet_b200.quantized_cache_read(state['cache'], state['slots'], state['dtype'])
        if kind == 'attention':
            return hidet_b200.quantized_cache_attention(state['q'], state['cache'], state['table'], state['lengths'], starts=state['starts'],
                                                        mask=state['mask'], return_lse=True)
        return hidet_b200.token_log_probs(state['logits'], state['tokens'], top=state['top'])
    if kind == 'rotary':
        return tuple(_rotated(state[n], state['positions'], state['table'], state['layout']).to(state[n].dtype) for n in ('q', 'k'))
    if kind == 'append':
        q, k = (_rotated(state[n], state['positions'], state['table'], state['layout']) for n in ('q', 'k'))
        _write(state['cache'], state['slots'], k, state['v'].float(), state['dim'])
        return (q.to(state['dtype']),) + tuple(x.to(state['dtype']) for x in _rows_of(state['cache'], state['slots'], state['dim']))
    if kind == 'read':
        return tuple(x.to(state['dtype']) for x in _rows_of(state['cache'], state['slots'], state['dim']))
    if kind == 'attention':
        return _plain_attention(state)
    return _plain_log_probs(state['logits'], state['tokens'], state['top'])


# ---- exact ----

def _exact_rotated(x, positions, table, layout):
    """Every pair of elements as a complex number, turned by its angle."""
    x, half = x.double(), table.shape[1] // 2
    turn = torch.complex(table[positions, :half].double(), table[positions, half:].double())[:, None]
    pairs = x[..., :2 * half].unflatten(-1, (2, half) if layout == 'half' else (half, 2))
    pairs = torch.view_as_complex((pairs.transpose(-1, -2) if layout == 'half' else pairs).contiguous()) * turn
    pairs = torch.view_as_real(pairs)
    y = x.clone()
    y[..., :2 * half] = (pairs.transpose(-1, -2) if layout == 'half' else pairs).flatten(-2)
    return y


def _exact_restored(x):
    x = x.double()
    step = x.abs().amax(-1, keepdim=True) / 127
    return torch.where(step > 0, torch.round(x / step) * step, 0.0)


def _exact_cached(cache, table_row, length, head, dim):
    """K and V [length, dim] of one head of one sequence, byte by byte from the records."""
    record = cache[table_row.long(), head].flatten(0, 1)[:-(-length // 16)]          # [blocks, bytes]
    r, d = torch.arange(16, device=cache.device)[:, None], torch.arange(dim, device=cache.device)
    chunks = math.gcd(dim // 16, 8)
    out = []
    for i, rank in enumerate((4 * (r // 8 % 2) + 2 * (r // 4 % 2) + r % 2, r % 8)):
        place = i * 16 * dim + r * dim + 16 * ((d // 16) ^ (rank * chunks // 8)) + d % 16
        scale = record[:, 32 * dim + 64 * i:32 * dim + 64 * (i + 1)].contiguous().view(torch.float32).double()
        out.append(((record[:, place].double() - 128) * scale[..., None]).flatten(0, 1)[:length])
    return out


def exact(case, seed):
    state = prepare(case, seed)
    kind = case['kind']
    if kind == 'rotary':
        return tuple(_exact_rotated(state[n], state['positions'], state['table'], state['layout']) for n in ('q', 'k'))
    if kind == 'append':
        q, k = (_exact_rotated(state[n], state['positions'], state['table'], state['layout']) for n in ('q', 'k'))
        return q, _exact_restored(k), _exact_restored(state['v'])
    if kind == 'read':
        page_size, dim = case['page_size'], case['dim']
        pages = state['slots'][::page_size] // page_size
        both = [_exact_cached(state['cache'], pages, case['tokens'], h, dim) for h in range(case['kv_heads'])]
        return tuple(torch.stack([x[i] for x in both], 1) for i in (0, 1))
    if kind == 'attention':
        tokens, lengths, dim = _tokens(case), _lengths(case), case['dim']
        group = case['heads'] // case['kv_heads']
        out = torch.empty(state['q'].shape, dtype=torch.float64, device='cuda')
        lse = torch.empty(state['q'].shape[:2], dtype=torch.float64, device='cuda')
        first = 0
        for b, (t, n) in enumerate(zip(tokens, lengths)):
            seen = torch.ones((t, n), dtype=torch.bool, device='cuda')
            if case['tree']:
                seen[:, n - t:] = state['mask'][first:first + t, :t]
            for h in range(case['kv_heads']):
                k, v = _exact_cached(state['cache'], state['table'][b], n, h, dim)
                q = state['q'][first:first + t, h * group:(h + 1) * group].double()
                s = torch.einsum('tgd,nd->tgn', q, k) / math.sqrt(dim)
                s = torch.where(seen[:, None], s, -math.inf)
                total = torch.logsumexp(s, -1)
                out[first:first + t, h * group:(h + 1) * group] = torch.einsum('tgn,nd->tgd', (s - total[..., None]).exp(), v)
                lse[first:first + t, h * group:(h + 1) * group] = total
            first += t
        return out, lse
    x = state['logits'].double()
    log_p = torch.log_softmax(x, -1)
    entropy = -(log_p.exp() * log_p).sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :case['top']]
    return log_p.gather(1, state['tokens']), entropy, log_p.gather(1, order), order
