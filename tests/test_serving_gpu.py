"""Rotary positions, the quantized cache, attention over it and token log probabilities against their definitions in 64 bits."""
import math

import pytest
import torch

import hidet_b200
from hidet_b200 import ffi
from serving_reference import TINY, U, attention, cached, log_probs, rotary

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def normal(*shape, seed=0, dtype=torch.float16, std=1.0):
    return (torch.randn(shape, device='cuda', generator=torch.Generator('cuda').manual_seed(seed)) * std).to(dtype)


def status():
    return ffi.func('b200q_check_status')()


@pytest.fixture(autouse=True)
def clean_status():
    yield
    assert status() == ffi.OK


def reported(match):
    with pytest.raises(ffi.BackendException, match=match):
        status()


def within(got, want, bound):
    got = got.double()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    off = (got - want).abs()[fine]
    over = (off - bound.expand(want.shape)[fine])
    assert not len(over) or over.max() <= 0, 'off by {:.3g}, {:.3g} more than allowed'.format(off.max().item(), over.max().item())


# ---------------------------------------------------------------------------------------------------------------- rotary

@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('tokens,heads,kv_heads,dim,rotary_dim', [(1, 32, 32, 128, 128), (5, 4, 1, 64, 32), (77, 3, 2, 80, 20), (3, 1, 1, 2, 2), (300, 8, 2, 96, 96),
                                                                  (9, 7, 0, 128, 64), (2, 5, 3, 33, 6), (1100, 5, 1, 256, 256)])
def test_rotary(dtype, layout, tokens, heads, kv_heads, dim, rotary_dim):
    table = hidet_b200.rotary_table(2000, rotary_dim)
    q, k = normal(tokens, heads, dim, dtype=dtype), normal(tokens, kv_heads, dim, dtype=dtype, seed=1) if kv_heads else None
    positions = torch.randint(0, 2000, (tokens,), device='cuda', generator=torch.Generator('cuda').manual_seed(2))
    a, b = hidet_b200.rotary_embedding(q, k, positions, table, layout=layout)
    within(a, *rotary(q, positions, table, layout))
    if k is None:
        assert b is None
    else:
        within(b, *rotary(k, positions, table, layout))
    assert torch.equal(a[..., rotary_dim:], q[..., rotary_dim:])


@pytest.mark.parametrize('dtype', TYPES)
def test_rotary_of_views_in_place_and_of_other_shapes(dtype):
    table = hidet_b200.rotary_table(512, 64)
    rows = normal(2, 33, 6 * 64 + 8, dtype=dtype)
    positions = (torch.arange(66, device='cuda').reshape(2, 33) * 7).to(torch.int32)
    for first in (0, 8, 1):  # aligned views, and one that is not
        qkv = rows[..., first:first + 6 * 64].unflatten(-1, (6, 64))
        q, k = qkv[..., :4, :], qkv[..., 4:5, :]
        want = hidet_b200.rotary_embedding(q.contiguous().flatten(0, 1), k.contiguous().flatten(0, 1), positions.flatten().long(), table)
        got = hidet_b200.rotary_embedding(q, k, positions, table)
        assert all(torch.equal(x.flatten(0, 1), y) for x, y in zip(got, want))
    before = rows.clone()
    qkv = rows[..., :6 * 64].unflatten(-1, (6, 64))
    q, k = qkv[..., :4, :], qkv[..., 4:5, :]
    want = hidet_b200.rotary_embedding(q, k, positions, table)
    got = hidet_b200.rotary_embedding(q, k, positions, table, out=(q, k))
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(rows[..., 5 * 64:], before[..., 5 * 64:])


def test_rotary_of_nothing_and_outside_the_table():
    table = hidet_b200.rotary_table(16, 64)
    q = normal(4, 3, 64)
    assert hidet_b200.rotary_embedding(q[:0], None, torch.zeros(0, dtype=torch.int64, device='cuda'), table)[0].shape == (0, 3, 64)
    positions = torch.tensor([3, 16, -1, 15], device='cuda')
    got, _ = hidet_b200.rotary_embedding(q, None, positions, table)
    within(got, *rotary(q, positions, table, 'half'))
    assert not got[1:3].any()
    reported('a position outside a rotary table')
    odd = normal(4, 3, 30)
    got, _ = hidet_b200.rotary_embedding(odd, None, positions, table[:, :10].contiguous())
    assert not got[1:3, :, :10].any() and torch.equal(got[1:3, :, 10:], odd[1:3, :, 10:])
    reported('a position outside a rotary table')


def test_rotary_tables():
    plain = hidet_b200.rotary_table(4096, 64)
    assert plain.dtype == torch.float32 and plain.shape == (4096, 64)
    assert torch.equal(hidet_b200.rotary_table(4096, 64, scaling='linear', factor=4.0)[::4], plain[:1024])
    ntk = hidet_b200.rotary_table(4096, 64, scaling='ntk', factor=4.0)
    angle = 4000 * (10000.0 * 4.0 ** (64 / 62)) ** (-62 / 64)
    assert abs(ntk[4000, 31].item() - math.cos(angle)) < 1e-6 and abs(angle - 1000 * 10000.0 ** (-62 / 64)) < 1e-9
    by = 0.1 * math.log(4.0) + 1.0
    yarn = hidet_b200.rotary_table(4096, 64, scaling='yarn', factor=4.0)
    assert torch.allclose(yarn[:, 0], plain[:, 0] * by, atol=1e-6) and torch.allclose(yarn[::4, 31], plain[:1024, 31] * by, atol=1e-6)
    with pytest.raises(ValueError, match='even'):
        hidet_b200.rotary_table(16, 7)
    with pytest.raises(ValueError, match='scaling'):
        hidet_b200.rotary_table(16, 8, scaling='more')


# ----------------------------------------------------------------------------------------------------------------- cache

def slots_of(n, total, seed=3, dtype=torch.int64):
    return torch.randperm(total, device='cuda', generator=torch.Generator('cuda').manual_seed(seed))[:n].to(dtype)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('tokens,kv_heads,dim,page_size', [(1, 1, 128, 64), (50, 3, 64, 16), (7, 2, 96, 48), (200, 1, 192, 32), (33, 5, 256, 128), (700, 8, 128, 16)])
def test_cache_rows_come_back_as_documented(dtype, tokens, kv_heads, dim, page_size):
    pages = -(-tokens // page_size) + 2
    cache = hidet_b200.quantized_cache(pages, kv_heads, dim, page_size)
    k, v = normal(tokens, kv_heads, dim, dtype=dtype, seed=4), normal(tokens, kv_heads, dim, dtype=dtype, seed=5, std=30.0)
    slots = slots_of(tokens, pages * page_size)
    assert hidet_b200.quantized_cache_append(cache, k, v, slots) is None
    back = hidet_b200.quantized_cache_read(cache, slots, torch.float32)
    for x, y in zip((k, v), back):
        codes, scales = cached(x)
        assert torch.equal(y, codes * scales[..., None])
        assert ((y.double() - x.double()).abs() <= scales.double()[..., None] * (0.5 + 2.0 ** -14)).all()
    for other in (torch.float16, torch.bfloat16):
        assert all(torch.equal(x.to(other), y) for x, y in zip(back, hidet_b200.quantized_cache_read(cache, slots.to(torch.int32), other)))
    rest = torch.ones(pages * page_size, dtype=torch.bool, device='cuda')
    rest[slots] = False
    empty = hidet_b200.quantized_cache_read(cache, rest.nonzero()[:, 0], torch.float32)
    assert not empty[0].any() and not empty[1].any()


@pytest.mark.parametrize('dtype', TYPES)
def test_cache_of_special_rows(dtype):
    x = torch.zeros(8, 1, 64, dtype=torch.float32)
    x[1] = -1.5
    x[2, 0, 3] = 1e-7 if dtype == torch.float16 else 1e-29
    x[3, 0, 5] = math.nan
    x[4, 0, 60] = -math.inf
    x[5, 0, :] = torch.finfo(dtype).max
    x[6, 0, 1] = -torch.finfo(dtype).max
    x[7, 0, ::2] = 127.0
    x[7, 0, 1::2] = torch.arange(32) + 0.5  # ties
    x = x.to(dtype).cuda()
    cache = hidet_b200.quantized_cache(1, 1, 64, 16)
    slots = torch.arange(8, device='cuda')
    hidet_b200.quantized_cache_append(cache, x, x, slots)
    for y in hidet_b200.quantized_cache_read(cache, slots, torch.float32):
        codes, scales = cached(x)
        assert torch.equal(y.nan_to_num(nan=-7.0), (codes * scales[..., None]).nan_to_num(nan=-7.0))
        assert not y[0].any() and y[3].isnan().all() and y[4].isnan().all()
    if dtype != torch.float16:
        tiny = torch.full((1, 1, 64), 1e-36, dtype=dtype, device='cuda')
        hidet_b200.quantized_cache_append(cache, tiny, tiny, slots[:1])
        assert not hidet_b200.quantized_cache_read(cache, slots[:1])[0].any()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('tokens,heads,kv_heads,dim,rotary_dim', [(1, 32, 32, 128, 128), (19, 4, 2, 64, 32), (130, 6, 3, 96, 96), (5, 2, 1, 192, 64), (40, 8, 1, 256, 256), (3000, 4, 1, 128, 64)])
def test_append_rotates_on_the_way(dtype, layout, tokens, heads, kv_heads, dim, rotary_dim):
    table = hidet_b200.rotary_table(4000, rotary_dim, scaling='yarn', factor=2.0)
    qkv = normal(tokens, heads + 2 * kv_heads, dim, dtype=dtype, seed=6)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], 1)
    positions = torch.randint(0, 4000, (tokens,), device='cuda', generator=torch.Generator('cuda').manual_seed(7)).to(torch.int32)
    cache = hidet_b200.quantized_cache(-(-tokens // 64) + 1, kv_heads, dim)
    slots = slots_of(tokens, cache.shape[0] * 64, dtype=torch.int32)
    got = hidet_b200.quantized_cache_append(cache, k, v, slots, q=q, positions=positions, table=table, layout=layout)
    assert torch.equal(got, hidet_b200.rotary_embedding(q, None, positions, table, layout=layout)[0])
    back_k, back_v = hidet_b200.quantized_cache_read(cache, slots, torch.float32)
    turned = hidet_b200.rotary_embedding(k.float(), None, positions, table, layout=layout)[0]
    for x, y in ((turned, back_k), (v, back_v)):
        codes, scales = cached(x)
        assert torch.equal(y, codes * scales[..., None])
    without = torch.zeros_like(cache)
    assert hidet_b200.quantized_cache_append(without, k, v, slots, positions=positions, table=table, layout=layout) is None
    assert torch.equal(without, cache)


def test_append_of_unaligned_rows_and_other_shapes():
    rows = normal(2, 9, 3 * 64 + 1, seed=8)
    table = hidet_b200.rotary_table(64, 64)
    positions = torch.arange(18, device='cuda').reshape(2, 9)
    q, k, v = (rows[..., 1 + 64 * i:65 + 64 * i].unflatten(-1, (1, 64)) for i in range(3))
    caches = [hidet_b200.quantized_cache(2, 1, 64, 16) for _ in range(2)]
    a = hidet_b200.quantized_cache_append(caches[0], k, v, positions + 3, q=q, positions=positions, table=table)
    b = hidet_b200.quantized_cache_append(caches[1], *(x.flatten(0, 1).contiguous() for x in (k, v)), positions.flatten() + 3,
                                          q=q.flatten(0, 1).contiguous(), positions=positions.flatten(), table=table)
    assert torch.equal(a.flatten(0, 1), b) and torch.equal(*caches) and caches[0].any()
    k2, v2 = hidet_b200.quantized_cache_read(caches[0], positions + 3)
    assert k2.shape == (2, 9, 1, 64) and torch.equal(v2.flatten(0, 1), hidet_b200.quantized_cache_read(caches[0], positions.flatten() + 3)[1])


def test_slots_that_are_padding_or_outside():
    cache = hidet_b200.quantized_cache(2, 2, 64, 16)
    k = normal(5, 2, 64, seed=9)
    slots = torch.tensor([31, -1, 32, 0, -5], device='cuda')
    hidet_b200.quantized_cache_append(cache, k[[0, 1, 3, 4]], k[[0, 1, 3, 4]], slots[[0, 1, 3, 4]])
    assert status() == ffi.OK
    back = hidet_b200.quantized_cache_read(cache, torch.arange(32, device='cuda'))[0]
    assert back[31].any() and back[0].any() and not back[1:31].any()
    before = cache.clone()
    hidet_b200.quantized_cache_append(cache, k, k, slots)
    reported('a slot outside a cache')
    assert torch.equal(cache, before)
    k2, v2 = hidet_b200.quantized_cache_read(cache, slots[[1, 0]])
    assert not k2[0].any() and not v2[0].any() and k2[1].any() and status() == ffi.OK
    k2, _ = hidet_b200.quantized_cache_read(cache, slots[2:3])
    assert not k2.any()
    reported('a slot outside a cache')
    table = hidet_b200.rotary_table(4, 64)
    hidet_b200.quantized_cache_append(cache, k[:1], k[:1], slots[:1], positions=torch.tensor([4], device='cuda'), table=table)
    reported('a position outside a rotary table')
    k2, v2 = hidet_b200.quantized_cache_read(cache, slots[:1])
    assert not k2.any() and v2.any()
    assert hidet_b200.quantized_cache_read(cache, slots[:0])[0].shape == (0, 2, 64)


# ------------------------------------------------------------------------------------------------------------- attention

def a_cache(lengths, kv_heads, dim, page_size, seed=10, std=1.0, v_std=1.0, spare=3):
    """A cache with random rows everywhere, and the table of pages of sequences of these lengths."""
    used = [-(-n // page_size) for n in lengths]
    cache = hidet_b200.quantized_cache(sum(used) + spare, kv_heads, dim, page_size)
    total = cache.shape[0] * page_size
    for first in range(0, total, 1 << 15):
        slots = torch.arange(first, min(total, first + (1 << 15)), device='cuda')
        hidet_b200.quantized_cache_append(cache, normal(len(slots), kv_heads, dim, seed=seed + first, std=std), normal(len(slots), kv_heads, dim, seed=seed + 1 + first, std=v_std), slots)
    order = torch.randperm(cache.shape[0], device='cuda', generator=torch.Generator('cuda').manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lengths), max(used + [1])), 2 ** 30, dtype=torch.int32, device='cuda')  # what is not used is not read
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    return cache, table


def slots_in(table, b, n, page_size):
    at = torch.arange(n, device='cuda')
    return table[b, at // page_size].long() * page_size + at % page_size


def check_attention(lengths, tokens, heads, kv_heads, dim, page_size, dtype, mask=None, std=1.0, scale=None, cache=None, q=None):
    cache, table = cache if cache is not None else a_cache(lengths, kv_heads, dim, page_size)
    starts = [sum(tokens[:b]) for b in range(len(tokens) + 1)]
    q = normal(sum(tokens), heads, dim, seed=11, dtype=dtype, std=std) if q is None else q
    n = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    out, lse = hidet_b200.quantized_cache_attention(q, cache, table, n, starts=torch.tensor(starts, dtype=torch.int32, device='cuda'), mask=mask, scale=scale, return_lse=True)
    assert out.shape == q.shape and out.dtype == dtype and lse.shape == q.shape[:2] and lse.dtype == torch.float32
    for b in range(len(lengths)):
        rows = slice(starts[b], starts[b + 1])
        if not tokens[b]:
            continue
        if lengths[b]:
            k, v = (x.double() for x in hidet_b200.quantized_cache_read(cache, slots_in(table, b, lengths[b], page_size), torch.float32))
        else:
            k = v = torch.zeros((0, kv_heads, dim), dtype=torch.float64, device='cuda')
        want, want_lse, bound, bound_lse = attention(q[rows], k, v, tokens[b], None if mask is None else mask[rows], 1 / math.sqrt(dim) if scale is None else scale)
        within(lse[rows], want_lse, bound_lse)
        within(out[rows], want, bound)
    return out, lse


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('heads,kv_heads,dim,page_size', [(4, 4, 128, 64), (8, 1, 128, 16), (5, 1, 64, 32), (24, 2, 128, 48), (6, 3, 96, 16), (2, 1, 192, 128), (16, 2, 256, 64), (64, 2, 64, 256)])
@pytest.mark.parametrize('length', [1, 15, 16, 17, 64, 65, 129, 1000])
def test_one_token(dtype, heads, kv_heads, dim, page_size, length):
    check_attention([length], [1], heads, kv_heads, dim, page_size, dtype)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('heads,kv_heads,dim', [(4, 4, 128), (16, 2, 128), (7, 1, 64), (8, 2, 96), (4, 1, 256), (4, 2, 192)])
def test_ragged_batches_of_several_tokens(dtype, heads, kv_heads, dim):
    lengths = [5, 700, 64, 1, 333, 130, 0, 2049, 40, 16]
    tokens = [5, 3, 64, 1, 17, 0, 2, 9, 33, 1]  # an empty cache with rows, a sequence without rows, more rows than positions
    check_attention(lengths, tokens, heads, kv_heads, dim, 16, dtype)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('heads,kv_heads,dim,most', [(4, 4, 128, 8), (16, 2, 128, 40), (32, 8, 64, 64), (8, 1, 96, 20), (4, 2, 256, 12), (8, 2, 128, 150)])
def test_trees_and_rows_that_see_nothing(dtype, heads, kv_heads, dim, most):
    tokens = [most, 1, most // 2, 3, most]
    lengths = [most + 500, 1, most // 2, 90, most + 31]
    mask = torch.rand((sum(tokens), most + 3), device='cuda', generator=torch.Generator('cuda').manual_seed(12)) < 0.4
    first = sum(tokens[:2])
    mask[first:first + most // 2] &= torch.arange(most // 2, device='cuda')[:, None] % 3 > 0  # a sequence of drafted tokens alone: rows that see nothing
    out, lse = check_attention(lengths, tokens, heads, kv_heads, dim, 32, dtype, mask=mask)
    assert lse[first].isinf().all() and not out[first].any()
    again = check_attention(lengths, tokens, heads, kv_heads, dim, 32, dtype, mask=mask.to(torch.uint8))
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


def test_more_columns_of_a_sequence_than_a_mask_has_are_not_seen():
    tokens, lengths = [6, 2], [50, 20]
    cache = a_cache(lengths, 2, 64, 16)
    mask = torch.ones((8, 6), dtype=torch.bool, device='cuda')
    mask[:, 4:] = False
    q = normal(8, 4, 64, seed=13)
    want = check_attention(lengths, tokens, 4, 2, 64, 16, torch.float16, mask=mask, cache=cache, q=q)[0]
    starts, n = (torch.tensor(x, dtype=torch.int32, device='cuda') for x in ([0, 6, 8], lengths))
    assert torch.equal(want, hidet_b200.quantized_cache_attention(q, cache[0], cache[1], n, starts=starts, mask=mask[:, :4]))


@pytest.mark.parametrize('length', [20000, 70001])
def test_long_contexts_and_large_scores(length):
    cache = a_cache([length], 1, 128, 64, std=3.0)
    for std, scale in ((1.0, None), (20.0, None), (0.01, 5.0)):
        check_attention([length], [1], 8, 1, 128, 64, torch.float16, cache=cache, std=std, scale=scale)
        check_attention([length], [1], 8, 1, 128, 64, torch.bfloat16, cache=cache, std=std, scale=scale)


def test_a_long_tail_of_small_probabilities_counts():
    """One position far above the others: 2^-20 of its probability each, together a tenth of the sum."""
    n, dim = 100000, 64
    cache = hidet_b200.quantized_cache(-(-n // 64), 1, dim, 64)
    k = torch.zeros((n, 1, dim), device='cuda')
    k[0, 0, 0] = 1.0
    v = torch.ones((n, 1, dim), device='cuda')
    v[0] = -1.0
    hidet_b200.quantized_cache_append(cache, k, v, torch.arange(n, device='cuda'))
    table = torch.arange(cache.shape[0], dtype=torch.int32, device='cuda')[None]
    q = torch.zeros((1, 1, dim), device='cuda', dtype=torch.float16)
    q[0, 0, 0] = 20 * math.log(2.0) * math.sqrt(dim)
    check_attention([n], [1], 1, 1, dim, 64, torch.float16, cache=(cache, table), q=q)


def test_values_of_any_size():
    lengths = [300]
    for v_std in (1e-4, 2000.0, 1e4):
        check_attention(lengths, [2], 4, 2, 128, 16, torch.bfloat16, cache=a_cache(lengths, 2, 128, 16, v_std=v_std))
    cache, table = a_cache(lengths, 2, 128, 16)
    rows = normal(300, 2, 128, dtype=torch.float32) * torch.logspace(-20, 20, 300, device='cuda')[:, None, None]
    hidet_b200.quantized_cache_append(cache, normal(300, 2, 128, dtype=torch.float32), rows, slots_in(table, 0, 300, 16))
    check_attention(lengths, [2], 4, 2, 128, 16, torch.bfloat16, cache=(cache, table))
    q = normal(2, 4, 128, dtype=torch.float32)
    for std in (1e30, 1e-30):
        check_attention(lengths, [2], 4, 2, 128, 16, torch.bfloat16, cache=(cache, table), q=(q * std).bfloat16(), scale=1e-20 if std > 1 else None)


def test_what_is_not_seen_does_not_matter():
    """NaN rows in positions behind the end, and in drafted positions that a row does not see."""
    lengths, tokens, page = [70, 9], [4, 4], 16
    cache, table = a_cache(lengths, 2, 64, page)
    mask = torch.tril(torch.ones((4, 4), dtype=torch.bool, device='cuda')).repeat(2, 1)
    q = normal(8, 4, 64, seed=14)
    n, starts = (torch.tensor(x, dtype=torch.int32, device='cuda') for x in (lengths, [0, 4, 8]))
    want = [hidet_b200.quantized_cache_attention(q, cache, table, n, starts=starts, mask=m) for m in (mask, None)]
    assert torch.equal(*want)
    bad = torch.full((1, 2, 64), math.nan, device='cuda')
    for b in range(2):
        behind = table[b, (lengths[b] - 1) // page].long() * page + torch.arange(lengths[b] % page, page, device='cuda')
        hidet_b200.quantized_cache_append(cache, bad.expand(len(behind), 2, 64), bad.expand(len(behind), 2, 64), behind)
        last = slots_in(table, b, lengths[b], page)[-1:]
        hidet_b200.quantized_cache_append(cache, bad, bad, last)  # only the last token sees this
    for m, w in zip((mask, None), want):
        got = hidet_b200.quantized_cache_attention(q, cache, table, n, starts=starts, mask=m)
        for b in range(2):
            assert torch.equal(got[4 * b:4 * b + 3], w[4 * b:4 * b + 3]) and got[4 * b + 3].isnan().all()
    q[5] = math.nan
    got = hidet_b200.quantized_cache_attention(q, cache, table, n, starts=starts)
    assert got[5].isnan().all() and torch.equal(got[4], want[1][4]) and torch.equal(got[:3], want[1][:3])


def test_forms_of_the_query():
    lengths = [100, 40, 77]
    cache, table = a_cache(lengths, 2, 64, 16)
    n = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    q = normal(3, 5, 4, 64, seed=15)
    starts = torch.tensor([0, 5, 10, 15], dtype=torch.int32, device='cuda')
    want, lse = hidet_b200.quantized_cache_attention(q.flatten(0, 1), cache, table, n, starts=starts, return_lse=True)
    got, got_lse = hidet_b200.quantized_cache_attention(q, cache, table, n, return_lse=True)
    assert torch.equal(got, want.unflatten(0, (3, 5))) and torch.equal(got_lse, lse.unflatten(0, (3, 5)))
    one = q[:, 0]
    want = hidet_b200.quantized_cache_attention(one.contiguous(), cache, table, n)
    assert torch.equal(hidet_b200.quantized_cache_attention(one, cache, table, n), want)                      # strides between tokens
    wide = normal(3, 4 * 64 + 1)
    wide[:, 1:] = one.flatten(1)
    assert torch.equal(hidet_b200.quantized_cache_attention(wide[:, 1:].unflatten(1, (4, 64)), cache, table, n), want)  # and no alignment
    assert torch.equal(hidet_b200.quantized_cache_attention(one, cache, table.repeat(1, 2)[:, :table.shape[1]], n), want)
    assert hidet_b200.quantized_cache_attention(q[:0, 0], cache, table[:0], n[:0]).shape == (0, 4, 64)


def test_lengths_and_pages_outside_are_reported_and_harmless():
    lengths = [100, 40]
    cache, table = a_cache(lengths, 1, 64, 16)
    q = normal(2, 2, 64, seed=16)
    n = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    want = hidet_b200.quantized_cache_attention(q, cache, table, n)
    whole = table.shape[1] * 16
    got = hidet_b200.quantized_cache_attention(q, cache, table, torch.tensor([10 ** 6, 40], dtype=torch.int32, device='cuda'))
    reported('a length beyond its page table')
    assert torch.equal(got[1], want[1])
    assert torch.equal(got[0], hidet_b200.quantized_cache_attention(q, cache, table, torch.tensor([whole, 40], dtype=torch.int32, device='cuda'))[0])
    for bad in (-1, cache.shape[0]):
        wrong = table.clone()
        wrong[0, 2] = bad
        got = hidet_b200.quantized_cache_attention(q, cache, wrong, n)
        reported('a page outside a cache')
        assert torch.equal(got[1], want[1]) and got.isfinite().all()
    got = hidet_b200.quantized_cache_attention(q, cache, table, torch.tensor([-3, 40], dtype=torch.int32, device='cuda'))
    assert not got[0].any() and torch.equal(got[1], want[1])


def test_results_do_not_depend_on_what_else_is_in_the_batch_order_or_run():
    """Sums are added in a fixed order: the same call gives the same bits."""
    lengths = [3000 + 17 * i for i in range(20)]
    cache, table = a_cache(lengths, 2, 128, 64)
    n = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    q = normal(20, 8, 128, seed=17)
    first = hidet_b200.quantized_cache_attention(q, cache, table, n)
    for _ in range(20):
        assert torch.equal(first, hidet_b200.quantized_cache_attention(q, cache, table, n))


def test_long_caches_pass_32_bits():
    """The last pages of a cache of more than 2^32 bytes."""
    page, dim = 64, 128
    pages = (1 << 32) // (page // 16 * (32 * dim + 128)) + 200
    cache = torch.empty((pages, 1, page // 16, 32 * dim + 128), dtype=torch.uint8, device='cuda')
    cache[-8:].zero_()
    small = torch.zeros_like(cache[-8:])
    k, v = normal(500, 1, dim, seed=18), normal(500, 1, dim, seed=19)
    slots = torch.arange(500, device='cuda')
    hidet_b200.quantized_cache_append(small, k, v, slots)
    hidet_b200.quantized_cache_append(cache, k, v, slots + (pages - 8) * page)
    assert torch.equal(cache[-8:], small)
    assert torch.equal(hidet_b200.quantized_cache_read(cache, slots + (pages - 8) * page)[1], hidet_b200.quantized_cache_read(small, slots)[1])
    table, n = torch.arange(8, dtype=torch.int32, device='cuda')[None], torch.tensor([500], dtype=torch.int32, device='cuda')
    q = normal(1, 4, dim, seed=20)
    assert torch.equal(hidet_b200.quantized_cache_attention(q, cache, table + (pages - 8), n), hidet_b200.quantized_cache_attention(q, small, table, n))


# ------------------------------------------------------------------------------------------------------------- log probs

def check_log_probs(logits, tokens, top):
    got = hidet_b200.token_log_probs(logits, tokens, top)
    lead = logits.shape[:-1]
    tk = tokens if tokens.dim() > len(lead) else tokens[..., None]
    (lp, entropy, values, order), (d, dh) = log_probs(logits, tk, top)
    assert got[0].shape == tokens.shape and [x.dtype for x in got] == [torch.float32] * 3 + [torch.int64]
    within(got[0].reshape(lp.shape), lp, d)
    within(got[1], entropy, dh)
    assert torch.equal(got[3], order)
    within(got[2], values, d)
    return got


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,vocab,given,top', [(1, 32000, 1, 5), (3, 7, 2, 7), (5, 1, 1, 1), (40, 513, 1, 32), (2, 32002, 4, 20), (7, 1500, 3, 32), (500, 4099, 1, 10), (1, 151936, 1, 20),
                                                  (9, 100003, 1, 32), (2, 250000, 600, 3), (300, 40000, 1, 0), (64, 64, 1, 1)])
def test_log_probs(dtype, rows, vocab, given, top):
    logits = normal(rows, vocab, seed=21, std=3.0, dtype=dtype)
    tokens = torch.randint(0, vocab, (rows, given), device='cuda', generator=torch.Generator('cuda').manual_seed(22))
    check_log_probs(logits, tokens, top)
    if given == 1:
        check_log_probs(logits, tokens[:, 0].to(torch.int32), top)


@pytest.mark.parametrize('dtype', TYPES)
def test_log_probs_with_ties_and_masked_tokens(dtype):
    vocab = 20000
    rows = torch.zeros((8, vocab), device='cuda')
    rows[1] = torch.arange(vocab, device='cuda') % 3
    rows[2, 5000:] = -math.inf
    rows[3] = -math.inf
    rows[3, [17, 19000, 4]] = torch.tensor([1.0, 1.0, -2.0], device='cuda')
    rows[4] = torch.linspace(-8, 8, vocab, device='cuda')
    rows[5] = -rows[4]
    rows[6, ::512 * 8] = 5.0
    rows[7] = normal(vocab, dtype=torch.float32).sign() * 0.0  # zeros of either sign are equal
    rows = rows.to(dtype)
    tokens = torch.full((8, 2), 17, device='cuda')
    tokens[:, 1] = vocab - 1
    for top in (1, 20, 32):
        check_log_probs(rows, tokens, top)
    for first in (1, 3):  # rows that start between two 16-byte boundaries, in one CTA and in several
        view = torch.zeros((8, vocab + 7), dtype=dtype, device='cuda')[:, first:first + vocab]
        view.copy_(rows)
        check_log_probs(view, tokens, 32)
        check_log_probs(view[4:5], tokens[4:5], 32)


def test_log_probs_when_one_thread_has_all_the_large_ones():
    """Candidates beyond what the list holds: the slower way gives the same."""
    vocab = 512 * 8 * 7 + 100
    rows = normal(3, vocab, seed=23, dtype=torch.float32)
    at = torch.arange(vocab, device='cuda')
    for thread in range(32):  # all elements of 32 threads of a CTA stand out
        rows[0, (at // 4) % 512 == thread] += 100.0
    rows[1] += 50.0 * ((at // 4) % 512 < 40)
    tokens = torch.zeros((3,), dtype=torch.int64, device='cuda')
    check_log_probs(rows.repeat(100, 1), tokens.repeat(100), 32)
    check_log_probs(rows, tokens, 32)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,vocab', [(6, 5000), (6, 200000)])
def test_log_probs_of_rows_without_a_distribution(dtype, rows, vocab):
    x = normal(rows, vocab, seed=24, dtype=dtype)
    x[1, 77] = math.nan
    x[2, vocab - 1] = math.inf
    x[3] = -math.inf
    x[4, :] = -math.inf
    x[4, vocab // 2] = 3.0
    tokens = torch.full((rows,), vocab // 2, device='cuda')
    got = hidet_b200.token_log_probs(x, tokens, top=4)
    for i in (1, 2, 3):
        assert got[0][i].isnan() and got[1][i].isnan() and got[2][i].isnan().all()
        assert ((got[3][i] >= 0) & (got[3][i] < vocab)).all()
    assert got[3][1, 0] == 77 and got[3][2, 0] == vocab - 1 and got[3][3].tolist() == [0, 1, 2, 3]
    assert got[0][4] == 0 and got[1][4] == 0 and got[3][4].tolist() == [vocab // 2, 0, 1, 2] and got[2][4, 1:].isinf().all()
    check_log_probs(x[[0, 4, 5]], tokens[[0, 4, 5]], 4)


def test_tokens_outside_the_vocabulary():
    x = normal(2, 100, seed=25)
    got = hidet_b200.token_log_probs(x, torch.tensor([100, 5], device='cuda'))
    reported('a token outside the vocabulary')
    assert got[0][0] == -math.inf and got[0][1].isfinite() and got[2].shape == (2, 0)
    assert hidet_b200.token_log_probs(x[:0], torch.zeros((0, 3), dtype=torch.int64, device='cuda'), 2)[2].shape == (0, 2)
    one = hidet_b200.token_log_probs(x[0], torch.tensor(5, device='cuda'), 2)
    assert one[0].shape == () and one[3].shape == (2,)
    check_log_probs(normal(2, 3, 50, seed=26), torch.zeros((2, 3), dtype=torch.int64, device='cuda'), 5)


# -------------------------------------------------------------------------------------------------------------- refusals

def test_refusals():
    cuda = dict(device='cuda')
    table, q = hidet_b200.rotary_table(16, 64), normal(2, 4, 64)
    at = torch.zeros(2, dtype=torch.int64, **cuda)
    cache, pages = hidet_b200.quantized_cache(4, 2, 64, 16), torch.zeros((2, 2), dtype=torch.int32, **cuda)
    n = torch.ones(2, dtype=torch.int32, **cuda)
    rot, app, read, att, lp = (getattr(hidet_b200, f) for f in ('rotary_embedding', 'quantized_cache_append', 'quantized_cache_read', 'quantized_cache_attention', 'token_log_probs'))
    kv = normal(2, 2, 64)
    for call, match in [
            (lambda: rot(q, None, at, table, layout='rows'), 'layout'), (lambda: rot(q, None, at[:1], table), 'positions'), (lambda: rot(q, None, at.float(), table), 'positions'),
            (lambda: rot(q, kv.bfloat16(), at, table), 'bfloat16'), (lambda: rot(q, None, at, table.half()), 'table'), (lambda: rot(q[..., :32], None, at, table), 'table'),
            (lambda: rot(q.to(torch.int8), None, at, table), 'float16, bfloat16'), (lambda: rot(q, kv[:1], at, table), 'k has shape'),
            (lambda: rot(q, kv, at, table, out=(q, None)), 'out'), (lambda: hidet_b200.quantized_cache(1, 1, 80), '80'), (lambda: hidet_b200.quantized_cache(1, 1, 64, 20), '20'),
            (lambda: app(cache, kv[:, :1], kv, at), 'k has shape'), (lambda: app(cache, kv, kv.bfloat16(), at), 'one type'), (lambda: app(cache, kv, kv, at[:1]), 'slots'),
            (lambda: app(cache, kv, kv, at, q=q), 'positions and a table'), (lambda: app(cache, kv, kv, at, positions=at), 'positions and a table'),
            (lambda: app(cache, kv, kv, at, positions=at, table=table[:, :24].contiguous()), 'multiples of 16'), (lambda: app(cache[:, :, :, 1:], kv, kv, at), 'cache'),
            (lambda: app(cache.float(), kv, kv, at), 'cache'), (lambda: read(cache, at, torch.int8), 'int8'), (lambda: read(cache, at.float()), 'slots'),
            (lambda: att(q.float(), cache, pages, n), 'float16 or bfloat16'), (lambda: att(q[:, :3], cache, pages, n), 'q has shape'), (lambda: att(q[..., :32], cache, pages, n), 'q has shape'),
            (lambda: att(q, cache, pages.long(), n), 'page table'), (lambda: att(q, cache, pages[:1], n), 'page table'), (lambda: att(q, cache, pages, n.long()), 'lengths'),
            (lambda: att(q[:1], cache, pages, n), 'rows of q'), (lambda: att(q, cache, pages, n, starts=n), 'starts'), (lambda: att(q, cache, pages, n, mask=n[:, None]), 'mask'),
            (lambda: att(q, cache, pages, n, mask=torch.zeros((2, 0), dtype=torch.bool, **cuda)), 'mask'),
            (lambda: lp(q[0], at, 1), 'tokens'), (lambda: lp(q[0, 0], at[0], 33), 'top'), (lambda: lp(q[0, 0, :3], at[0], 4), 'top'), (lambda: lp(at, at), 'float16, bfloat16')]:
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(ffi.BackendException, match='positive number'):
        att(q, cache, pages, n, scale=0.0)
    with pytest.raises(ffi.BackendException, match='positive number'):
        att(q, cache, pages, n, scale=math.nan)
    for call in (lambda: rot(q.cpu(), None, at, table), lambda: app(cache.cpu(), kv, kv, at), lambda: read(cache.cpu(), at), lambda: att(q, cache, pages.cpu(), n), lambda: lp(q[0].cpu(), at)):
        with pytest.raises(ffi.BackendException, match='CUDA devices only'):
            call()


def test_another_stream_and_a_graph():
    """Calls follow the current stream, and a captured step is replayed as its sequences grow."""
    kv_heads, dim, page = 2, 128, 16
    cache, pages = hidet_b200.quantized_cache(20, kv_heads, dim, page), torch.arange(20, dtype=torch.int32, device='cuda').reshape(2, 10)
    table = hidet_b200.rotary_table(200, dim)
    steps = 30
    qkv = normal(steps, 2, 8 + 2 * kv_heads, dim, seed=27)
    w = normal(8 * dim, 500, seed=28, std=0.05)

    def step(x, n, cache):
        q, k, v = x.split([8, kv_heads, kv_heads], 1)
        at = n.long() - 1
        slots = pages.gather(1, (at // page)[:, None])[:, 0].long() * page + at % page
        q = hidet_b200.quantized_cache_append(cache, k, v, slots, q=q, positions=at, table=table)
        out = hidet_b200.quantized_cache_attention(q, cache, pages, n)
        logits = out.flatten(1) @ w
        return [out] + list(hidet_b200.token_log_probs(logits, logits.argmax(-1), top=3))

    n = torch.zeros(2, dtype=torch.int32, device='cuda')
    want = []
    for i in range(steps):
        n += 1
        want.append([x.clone() for x in step(qkv[i], n, cache)])
    other = torch.cuda.Stream()
    cache2 = torch.zeros_like(cache)
    n.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        for i in range(steps):
            n += 1
            assert all(torch.equal(a, b) for a, b in zip(want[i], step(qkv[i], n, cache2)))
    other.synchronize()
    assert torch.equal(cache, cache2)
    cache2.zero_()
    x, n1 = qkv[0].clone(), torch.ones(2, dtype=torch.int32, device='cuda')
    graph = hidet_b200.CudaGraph(lambda: [x, n1], lambda inputs: step(inputs[0], inputs[1], cache2), ref_objs=[cache2])
    cache2.zero_()
    for i in range(steps):
        got = graph.run_async([qkv[i], torch.full((2,), i + 1, dtype=torch.int32, device='cuda')])
        assert all(torch.equal(a, b) for a, b in zip(want[i], got))
