"""The decoding operators on the ways through the code that a call takes seldom: the kernel for many rows on small sequences, the lists of the
log probabilities when they overflow, the Python path beside the native one, and all of them together in the example."""
import math

import pytest
import torch

import bench_decoder
import hidet_b200
from examples import tree_decoding
from hidet_b200 import ffi, native
from test_native_gpu import _both
from test_serving_gpu import TYPES, a_cache, check_attention, check_log_probs, clean_status, normal, slots_in  # noqa: F401

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------------------- attention of many rows

def wide(cache):
    """The page table as it is for sequences that may become long: this is what the kernel for many rows is chosen by."""
    pages, table = cache
    return pages, torch.cat([table, torch.full((table.shape[0], 40000), 2 ** 30, dtype=torch.int32, device='cuda')], 1)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('heads,kv_heads,dim,page_size', [(16, 2, 128, 16), (7, 1, 64, 48), (32, 8, 128, 64), (40, 8, 64, 256)])
def test_ragged_batches(dtype, heads, kv_heads, dim, page_size):
    lengths = [5, 700, 64, 1, 333, 130, 0, 2049, 40, 16]
    tokens = [5, 30, 64, 1, 17, 0, 2, 9, 70, 1]  # an empty cache with rows, a sequence without rows, more rows than positions
    check_attention(lengths, tokens, heads, kv_heads, dim, page_size, dtype, cache=wide(a_cache(lengths, kv_heads, dim, page_size)))


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('heads,kv_heads,dim,page_size', [(12, 3, 64, 16), (20, 4, 96, 48), (8, 2, 128, 64), (12, 3, 192, 16), (4, 1, 256, 256)])
def test_items_of_sixteen_rows(dtype, heads, kv_heads, dim, page_size):
    """Nine to sixteen rows a key/value head on average, much work by the page table."""
    lengths, tokens = [700, 64, 1, 333, 0, 2049, 16], [3, 4, 1, 9, 2, 3, 2]
    cache = wide(a_cache(lengths, kv_heads, dim, page_size))
    check_attention(lengths, tokens, heads, kv_heads, dim, page_size, dtype, cache=cache)
    mask = torch.rand((sum(tokens), 9), device='cuda', generator=torch.Generator('cuda').manual_seed(44)) < 0.5
    check_attention(lengths, tokens, heads, kv_heads, dim, page_size, dtype, cache=cache, mask=mask)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('heads,kv_heads,dim,most', [(16, 2, 128, 40), (8, 1, 64, 33), (32, 8, 128, 64), (4, 2, 128, 150)])
def test_trees(dtype, heads, kv_heads, dim, most):
    tokens = [most, 1, most // 2, 3, most]
    lengths = [most + 500, 1, most // 2, 90, most + 31]
    mask = torch.rand((sum(tokens), most + 3), device='cuda', generator=torch.Generator('cuda').manual_seed(42)) < 0.4
    first = sum(tokens[:2])
    mask[first:first + most // 2] &= torch.arange(most // 2, device='cuda')[:, None] % 3 > 0
    mask[:most] = torch.rand((most, most + 3), device='cuda', generator=torch.Generator('cuda').manual_seed(43)) < 0.05
    cache = wide(a_cache(lengths, kv_heads, dim, 32))
    out, lse = check_attention(lengths, tokens, heads, kv_heads, dim, 32, dtype, mask=mask, cache=cache)
    assert lse[first].isinf().all() and not out[first].any()
    narrow = torch.zeros((sum(tokens), most + 64), dtype=torch.uint8, device='cuda')[:, 5:5 + mask.shape[1]]  # rows that start anywhere
    narrow.copy_(mask)
    again = check_attention(lengths, tokens, heads, kv_heads, dim, 32, dtype, mask=narrow, cache=cache)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('dim', [64, 128])
def test_a_long_sequence_in_many_pieces(dtype, dim):
    lengths, tokens = [30001], [45]
    cache = wide(a_cache(lengths, 2, dim, 64, std=3.0))
    mask = torch.tril(torch.ones((45, 45), dtype=torch.bool, device='cuda'))
    for std, scale in ((1.0, None), (20.0, None), (0.01, 5.0)):
        want = check_attention(lengths, tokens, 10, 2, dim, 64, dtype, cache=cache, std=std, scale=scale)
        got = check_attention(lengths, tokens, 10, 2, dim, 64, dtype, cache=cache, std=std, scale=scale, mask=mask)
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_the_same_bits_whatever_ran_before():
    lengths, tokens = [3000 + 171 * i for i in range(6)], 24
    n = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    calls = []
    for dim in (64, 128):
        cache = wide(a_cache(lengths, 2, dim, 64))
        calls += [(normal(6, tokens, 8, dim, seed=17, dtype=dtype), *cache, n) for dtype in (torch.float16, torch.bfloat16)]
    first = [hidet_b200.quantized_cache_attention(*c) for c in calls]
    for _ in range(8):
        for c, want in zip(calls, first):
            assert torch.equal(want, hidet_b200.quantized_cache_attention(*c))


def test_values_of_any_size():
    lengths = [300, 80]
    for v_std in (1e-4, 2000.0, 1e4):
        check_attention(lengths, [40, 33], 4, 2, 128, 16, torch.bfloat16, cache=wide(a_cache(lengths, 2, 128, 16, v_std=v_std)))
    cache, table = wide(a_cache(lengths, 2, 128, 16))
    rows = normal(300, 2, 128, dtype=torch.float32) * torch.logspace(-20, 20, 300, device='cuda')[:, None, None]
    hidet_b200.quantized_cache_append(cache, normal(300, 2, 128, dtype=torch.float32), rows, slots_in(table, 0, 300, 16))
    check_attention(lengths, [40, 33], 4, 2, 128, 16, torch.bfloat16, cache=(cache, table))
    q = normal(73, 4, 128, dtype=torch.float32)
    for std in (1e30, 1e-30):
        check_attention(lengths, [40, 33], 4, 2, 128, 16, torch.bfloat16, cache=(cache, table), q=(q * std).bfloat16(), scale=1e-20 if std > 1 else None)


def test_what_is_not_seen_does_not_matter():
    """NaN rows in positions behind the end, and in drafted positions that a row does not see."""
    lengths, t, page = [300, 90], 40, 16
    cache, table = wide(a_cache(lengths, 2, 64, page))
    mask = torch.tril(torch.ones((t, t), dtype=torch.bool, device='cuda')).repeat(2, 1)
    q = normal(2, t, 4, 64, seed=14)
    n = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    want = hidet_b200.quantized_cache_attention(q, cache, table, n, mask=mask)
    assert torch.equal(want, hidet_b200.quantized_cache_attention(q, cache, table, n))
    bad = torch.full((1, 2, 64), math.nan, device='cuda')
    for b in range(2):
        behind = table[b, (lengths[b] - 1) // page].long() * page + torch.arange(lengths[b] % page, page, device='cuda')
        hidet_b200.quantized_cache_append(cache, bad.expand(len(behind), 2, 64), bad.expand(len(behind), 2, 64), behind)
        hidet_b200.quantized_cache_append(cache, bad, bad, slots_in(table, b, lengths[b], page)[-1:])  # only the last token sees this
    for m in (mask, None):
        got = hidet_b200.quantized_cache_attention(q, cache, table, n, mask=m)
        assert torch.equal(got[:, :-1], want[:, :-1]) and got[:, -1].isnan().all()
    q[1, 5] = math.nan
    got = hidet_b200.quantized_cache_attention(q, cache, table, n)
    assert got[1, 5].isnan().all() and torch.equal(got[1, 6:-1], want[1, 6:-1]) and torch.equal(got[0, :-1], want[0, :-1])


def test_lengths_and_pages_outside():
    lengths, t = [200, 100], 40
    cache, table = a_cache(lengths, 1, 64, 16)
    table = torch.cat([table, table[:1, :1].expand(2, 40000)], 1)
    q = normal(2, t, 8, 64, seed=16)
    n = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    want = hidet_b200.quantized_cache_attention(q, cache, table, n)
    for bad in (-1, cache.shape[0]):
        wrong = table.clone()
        wrong[0, 2] = bad
        got = hidet_b200.quantized_cache_attention(q, cache, wrong, n)
        with pytest.raises(ffi.BackendException, match='a page outside a cache'):
            ffi.func('b200q_check_status')()
        assert torch.equal(got[1], want[1]) and got.isfinite().all()
    got = hidet_b200.quantized_cache_attention(q, cache, table, torch.tensor([-3, 100], dtype=torch.int32, device='cuda'))
    assert not got[0].any() and torch.equal(got[1], want[1])


# ---------------------------------------------------------------------------------------------- log probabilities

@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [4096, 32002, 200000])
@pytest.mark.parametrize('hidden', ['infinity', 'lowest'])
def test_log_probs_of_few_allowed_tokens(dtype, vocab, hidden):
    """Rows with fewer allowed tokens than alternatives, and around that many: the others come by their index, with probability zero."""
    allowed = [1, 2, 5, 19, 20, 21, 40]
    rows = torch.full((len(allowed), vocab), -math.inf if hidden == 'infinity' else torch.finfo(dtype).min, dtype=dtype, device='cuda')
    gen = torch.Generator('cuda').manual_seed(31)
    for i, n in enumerate(allowed):
        rows[i, torch.randperm(vocab, device='cuda', generator=gen)[:n]] = normal(n, seed=32 + i, dtype=dtype)
    tokens = torch.randint(0, vocab, (len(allowed), 3), device='cuda', generator=gen)
    for top in (1, 20, 32):
        check_log_probs(rows, tokens, top)
        check_log_probs(rows.repeat(60, 1), tokens.repeat(60, 1), top)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [500, 32002, 200000])
def test_log_probs_of_rows_around_the_lowest_number(dtype, vocab):
    """The type's lowest number beside -inf, beside numbers a little larger, and alone."""
    low = torch.finfo(dtype).min
    rows = torch.full((5, vocab), -math.inf, dtype=dtype, device='cuda')
    rows[0, 7::9] = low
    rows[1] = low
    rows[2] = low
    rows[2, 3:400] = torch.linspace(1.0, 0.99, 397, device='cuda', dtype=torch.float64).mul(low).to(dtype)
    rows[3, vocab - 1] = low
    rows[4] = torch.linspace(low, 0.0, vocab, device='cuda', dtype=torch.float64).to(dtype)
    tokens = torch.tensor([[7, 8], [0, 1], [399, 2], [vocab - 1, 0], [vocab - 1, 0]], device='cuda')
    for top in (1, 32):
        check_log_probs(rows, tokens, top)
        check_log_probs(rows.repeat(60, 1), tokens.repeat(60, 1), top)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [600, 4096, 4200, 70001])
def test_log_probs_of_rows_with_few_different_values(dtype, vocab):
    gen = torch.Generator('cuda').manual_seed(33)
    rows = torch.stack([torch.full((vocab,), 1.5, device='cuda'), torch.randint(0, 2, (vocab,), device='cuda', generator=gen).float(),
                        torch.randint(0, 40, (vocab,), device='cuda', generator=gen).float() / 8, (torch.arange(vocab, device='cuda') > vocab - 9).float(),
                        (torch.arange(vocab, device='cuda') % 700 == 0) * 2.0]).to(dtype)
    tokens = torch.tensor([0, 1, 2, 3, vocab - 1], device='cuda')
    for top in (1, 7, 32):
        check_log_probs(rows, tokens, top)
        check_log_probs(rows.repeat(70, 1), tokens.repeat(70), top)


# --------------------------------------------------------------------------------------------- the two host paths

@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('lead', [(1,), (5,)])
def test_native_rotary_append_and_read(monkeypatch, dtype, layout, lead):
    assert native.load() is not None
    table = hidet_b200.rotary_table(50, 64)
    tokens = math.prod(lead)
    qkv = normal(*lead, 4 + 2 + 2, 64, seed=51, dtype=dtype)
    q, k, v = qkv.split([4, 2, 2], -2)
    at = torch.arange(3, 3 + tokens, device='cuda').reshape(lead)
    _both(monkeypatch, 'rotary', (q, k, at, table, layout), lambda: hidet_b200.rotary_embedding(q, k, at, table, layout=layout))
    caches = []
    for use in (True, False):
        cache = hidet_b200.quantized_cache(3, 2, 64, 16)
        with monkeypatch.context() as m:
            if not use:
                m.setattr(native, 'append', native._unavailable)
            rotated = hidet_b200.quantized_cache_append(cache, k, v, at, q=q, positions=at.to(torch.int32), table=table, layout=layout)
            assert hidet_b200.quantized_cache_append(cache, k, v, at + 20) is None
        caches.append((cache, rotated))
    direct = hidet_b200.quantized_cache(3, 2, 64, 16)
    rotated = native.append(direct, k, v, at, q, at.to(torch.int32), table, layout)
    assert native.append(direct, k, v, at + 20, None, None, None, 'half') is not None
    for cache, x in caches:
        assert torch.equal(cache, direct) and torch.equal(x, rotated) and x.shape == q.shape and x.dtype == dtype
    _both(monkeypatch, 'read', (direct, at, dtype), lambda: hidet_b200.quantized_cache_read(direct, at, dtype))


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
def test_native_attention(monkeypatch, dtype):
    lengths = [100, 40, 77]
    cache, table = a_cache(lengths, 2, 64, 16)
    n = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    starts = torch.tensor([0, 2, 9, 15], dtype=torch.int32, device='cuda')
    q = normal(15, 4, 64, seed=52, dtype=dtype)
    mask = torch.rand((15, 8), device='cuda', generator=torch.Generator('cuda').manual_seed(53)) < 0.5
    calls = [(q[:3], None, None), (q.unflatten(0, (3, 5)), None, mask), (q, starts, mask), (q, starts, None), (q[:, :2].contiguous(), starts, mask.to(torch.uint8))]
    for x, s, m in calls:
        for lse in (False, True):
            for scale in (None, 0.25):
                hidet_b200.quantized_cache_attention(x, cache, table, n, s, m)  # makes the stream's scratch
                _both(monkeypatch, 'attention', (x, cache, table, n, s, m, scale, lse),
                      lambda: hidet_b200.quantized_cache_attention(x, cache, table, n, starts=s, mask=m, scale=scale, return_lse=lse))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('lead,given', [((), None), ((3,), None), ((2, 3), None), ((3,), 4)])
def test_native_log_probs(monkeypatch, dtype, lead, given):
    x = normal(*lead, 333, seed=54, dtype=dtype)
    tokens = torch.randint(0, 333, lead + (() if given is None else (given,)), device='cuda', generator=torch.Generator('cuda').manual_seed(55))
    for t in (tokens, tokens.to(torch.int32)):
        for top in (0, 3):
            _both(monkeypatch, 'log_probs', (x, t, top), lambda: hidet_b200.token_log_probs(x, t, top))


def test_operands_the_native_path_leaves_to_the_python_path():
    """Among them tokens in two dimensions."""
    x, pos = normal(2, 3, 4, 64), torch.arange(6, device='cuda').reshape(2, 3)
    assert native.rotary(x, None, pos, hidet_b200.rotary_table(50, 64), 'half') is None
    both = [hidet_b200.rotary_embedding(y, None, p, hidet_b200.rotary_table(50, 64))[0] for y, p in ((x, pos), (x.flatten(0, 1), pos.flatten()))]
    assert torch.equal(both[0].flatten(0, 1), both[1])
    table, at = hidet_b200.rotary_table(50, 64), torch.zeros(2, dtype=torch.int64, device='cuda')
    q, kv, cache = normal(2, 4, 64), normal(2, 2, 64), hidet_b200.quantized_cache(3, 2, 64, 16)
    pages, n = torch.zeros((2, 2), dtype=torch.int32, device='cuda'), torch.ones(2, dtype=torch.int32, device='cuda')
    hidet_b200.quantized_cache_attention(q, cache, pages, n)
    for name, plain, others in [
            ('rotary', (q, kv, at, table, 'half'), [(0, q.cpu()), (0, q.double()), (1, kv.float()), (2, at.float()), (2, at[:1]), (3, table.half()), (3, table[:, :63]), (4, 'rows')]),
            ('append', (cache, kv, kv, at, q, at, table, 'half'), [(0, cache.float()), (0, cache[:, :, :, 1:]), (1, kv[:1]), (2, kv.float()), (3, at.short()), (4, q.float()), (5, at[:1]), (5, None), (6, table[:, :24]), (7, 0)]),
            ('read', (cache, at, torch.float16), [(0, cache.cpu()), (0, cache[:, :, :, 1:]), (1, at.float()), (1, at.cpu()), (2, torch.int8), (2, 'float16')]),
            ('attention', (q, cache, pages, n, None, None, None, False), [(0, q.float()), (0, q[:, :3]), (0, q[..., :32]), (0, q[:1]), (1, cache.cpu()), (2, pages.long()), (2, pages[:1]), (3, n.long()), (4, n), (5, n), (6, 'x')]),
            ('log_probs', (q[:, 0].contiguous(), at, 2), [(0, q[:, 0]), (0, q[:, 0].double()), (0, at), (1, at.float()), (1, at[:1]), (1, at.cpu()), (2, 33), (2, -1), (2, 'x')])]:
        assert getattr(native, name)(*plain) is not None, name
        for i, what in others:
            args = list(plain)
            args[i] = what
            assert getattr(native, name)(*args) is None, (name, i, what)


# -------------------------------------------------------------------------------------------------- all of them together

def test_tree_decoding_follows_the_decoder_in_32_bits():
    """The example's text, one token a pass and by trees, against the same decoder on dequantized weights in float32 that is fed that text.

    bench_decoder's int8 decoder may be off by 1 % of the largest logit (its own test).  A cached row's elements are off by up to 1 / 254 of its largest, about
    0.7 % of its root mean square each, for keys and for values and in each of three layers: 1 % more a layer at the most.  So 4 % of the largest logit,
    and twice that for a log probability, a difference of two such sums, and for the distance of the chosen token's from the best one's."""
    cfg, count = bench_decoder.SMALL, 40
    torch.manual_seed(7)
    with torch.device('cuda'):
        model = bench_decoder.Decoder(bench_decoder.DecoderConfig(cfg.vocab, cfg.hidden, cfg.heads, cfg.ffn, cfg.layers, cfg.prompt, count)).half().eval()
    prompt = torch.randint(0, cfg.vocab, (cfg.prompt,), device='cuda', generator=torch.Generator('cuda').manual_seed(7))
    with torch.no_grad():
        ref = bench_decoder.with_dequantized_weights(model).float()
        single = tree_decoding.TreeDecoding(model, cfg.prompt + count, rows=1).generate(prompt, count)
        assert single[2] == count - 1
        true = prompt.tolist() + single[0]

        def draft(text, rows):  # what comes next, each token beside wrong ones
            right = true[len(text):len(text) + 5] if text == true[:len(text)] else []
            return [right[:i] + [(right[i] + 1 + j) % cfg.vocab] for i in range(len(right)) for j in range(2)] + [right]

        known = tree_decoding.TreeDecoding(model, cfg.prompt + count, rows=16, draft=draft).generate(prompt, count, slack=1e-3)
        found = tree_decoding.TreeDecoding(model, cfg.prompt + count, rows=24).generate(prompt, count)
        for tokens, log_probs, passes in (single, known, found):
            assert len(tokens) == len(log_probs) == count and passes < count
            forced = [torch.tensor([t], device='cuda') for t in tokens]
            logits, _ = bench_decoder.greedy(ref, model.cfg, prompt[None], count - 1, forced=forced, dtype=torch.float32)
            want = torch.log_softmax(logits.double(), -1)
            own = want[torch.arange(count), torch.tensor(tokens)]
            tolerance = 2 * 0.04 * logits.abs().max().item()
            assert (torch.tensor(log_probs, device='cuda', dtype=torch.float64) - own).abs().max() <= tolerance
            assert (want.amax(-1) - own).max() <= tolerance
    if known[0] == single[0]:  # else a near tie sent them apart, within the bounds above
        assert known[2] <= count // 3
