"""The decoding operators where a call's data is at an end of its range: rows that no sequence has, and what their neighbours hold."""
import ctypes
import math

import pytest
import torch

import hidet_b200
from hidet_b200 import ffi
from hidet_b200.runtime import workspaces
from test_serving_gpu import TYPES, a_cache, check_attention, check_log_probs, clean_status, normal, slots_in  # noqa: F401
from test_serving_paths_gpu import wide

pytestmark = pytest.mark.gpu


def attention_into(out, lse, q, cache, table, lengths, starts=None, mask=None, mask_width=None):
    """The entry point's result in tensors of the caller's, contiguous q [tokens, heads, dim].  Returns them."""
    tokens, heads, dim = q.shape
    batch, kv_heads = len(lengths), cache.shape[1]
    need = ffi.func('b200q_quantized_cache_attention_workspace_bytes')(batch, tokens, heads, kv_heads, dim)
    workspace = torch.zeros(max(16, need), dtype=torch.uint8, device='cuda')
    ffi.func('b200q_quantized_cache_attention')(
        ctypes.byref(ffi.Heads(q.data_ptr(), heads * dim, dim)), out.data_ptr(), lse.data_ptr(), cache.data_ptr(), cache.shape[0], cache.shape[2] * 16, table.data_ptr(), table.shape[1],
        table.stride(0), lengths.data_ptr(), starts.data_ptr() if starts is not None else None, mask.data_ptr() if mask is not None else None,
        mask_width if mask_width is not None else mask.shape[1] if mask is not None else 0, mask.stride(0) if mask is not None else 0, batch, tokens, heads, kv_heads, dim, 1 / math.sqrt(dim),
        {torch.float16: ffi.F16, torch.bfloat16: ffi.BF16}[q.dtype], workspace.data_ptr(), workspace.numel(), torch.cuda.current_stream().cuda_stream)
    return out, lse


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device='cuda')


# heads, kv_heads, dim and tokens of two sequences, the page table made for long ones: one or two of 8 rows, of 16, and the kernel for many
FORMS = [(4, 2, 64, (1, 1), False), (4, 1, 128, (3, 5), False), (8, 1, 96, (2, 1), True), (8, 2, 128, (40, 23), True), (16, 2, 64, (9, 30), True)]


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('heads,kv_heads,dim,tokens,long', FORMS)
@pytest.mark.parametrize('front,behind', [(0, 3), (2, 0), (1, 700)])
def test_rows_that_no_sequence_has_are_zeros(dtype, heads, kv_heads, dim, tokens, long, front, behind):
    lengths = [700, 90]
    cache, table = a_cache(lengths, kv_heads, dim, 16)
    if long:
        cache, table = wide((cache, table))
    q = normal(front + sum(tokens) + behind, heads, dim, seed=61, dtype=dtype)
    starts, n = ints(front, front + tokens[0], front + sum(tokens)), ints(*lengths)
    out, lse = attention_into(torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device='cuda'), q, cache, table, n, starts)
    own = slice(front, front + sum(tokens))
    want = hidet_b200.quantized_cache_attention(q[own], cache, table, n, starts=starts - front, return_lse=True)
    if not behind == 700:  # so many rows may choose another kernel
        assert torch.equal(out[own], want[0]) and torch.equal(lse[own], want[1])
    for rest in (slice(0, front), slice(front + sum(tokens), None)):
        assert not out[rest].any() and (lse[rest] == -math.inf).all()


def test_rows_without_sequences():
    cache = hidet_b200.quantized_cache(2, 2, 64, 16)
    q = normal(5, 4, 64, seed=62)
    out, lse = hidet_b200.quantized_cache_attention(q, cache, ints().reshape(0, 3), ints(), starts=ints(0), return_lse=True)
    assert not out.any() and (lse == -math.inf).all()
    out, lse = attention_into(torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device='cuda'), q, cache, ints().reshape(0, 3), ints())
    assert not out.any() and (lse == -math.inf).all()
    out, lse = hidet_b200.quantized_cache_attention(q, cache, ints(0, 1)[:, None], ints(9, 4), starts=ints(2, 2, 2), return_lse=True)
    assert not out.any() and (lse == -math.inf).all()


@pytest.mark.parametrize('heads,kv_heads,dim,tokens,long', FORMS)
@pytest.mark.parametrize('starts', [(3, 1, 4), (0, 5, 4), (-1, 1, 2), (0, 1, 10 ** 6), (2 ** 31 - 1, 0, 2 ** 31 - 1), (0, 0, -2 ** 31)])
def test_starts_out_of_order_or_range_are_reported_and_harmless(heads, kv_heads, dim, tokens, long, starts):
    lengths = [700, 90]
    cache, table = a_cache(lengths, kv_heads, dim, 16)
    if long:
        cache, table = wide((cache, table))
    q, n = normal(sum(tokens) + 2, heads, dim, seed=63), ints(*lengths)
    out, lse = hidet_b200.quantized_cache_attention(q, cache, table, n, starts=ints(*starts), return_lse=True)
    with pytest.raises(ffi.BackendException, match='sequences whose rows are out of order or outside'):
        ffi.func('b200q_check_status')()
    assert not out.any() and (lse == -math.inf).all()
    fine = ints(0, tokens[0], sum(tokens))
    assert hidet_b200.quantized_cache_attention(q, cache, table, n, starts=fine)[:sum(tokens)].any()  # the workspace is as it was
    assert ffi.func('b200q_check_status')() == ffi.OK


@pytest.mark.parametrize('dim', [96, 128])
def test_sequences_that_all_claim_all_rows(dim):
    """More tiles together than 32 bits count."""
    cache = hidet_b200.quantized_cache(4, 8, dim, 64)
    q = normal(4096, 8, dim, seed=64)
    table = torch.zeros((64, 2048), dtype=torch.int32, device='cuda')
    n = torch.full((64,), 131072, dtype=torch.int32, device='cuda')
    out, lse = hidet_b200.quantized_cache_attention(q, cache, table, n, starts=ints(*[0, 4096] * 32, 0), return_lse=True)
    with pytest.raises(ffi.BackendException, match='sequences whose rows are out of order or outside'):
        ffi.func('b200q_check_status')()
    assert not out.any() and (lse == -math.inf).all()


@pytest.mark.parametrize('heads,kv_heads,dim,tokens,long', FORMS)
def test_a_width_without_a_mask_is_none(heads, kv_heads, dim, tokens, long):
    lengths = [700, 90]
    cache, table = a_cache(lengths, kv_heads, dim, 16)
    if long:
        cache, table = wide((cache, table))
    q = normal(sum(tokens), heads, dim, seed=65)
    starts, n = ints(0, tokens[0], sum(tokens)), ints(*lengths)
    want = hidet_b200.quantized_cache_attention(q, cache, table, n, starts=starts, return_lse=True)
    for width in (1, 64, 1 << 40):
        got = attention_into(torch.empty_like(q), torch.empty(q.shape[:2], device='cuda'), q, cache, table, n, starts, mask_width=width)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_wide_mask_of_a_very_long_sequence():
    """Positions and the mask's width together pass 31 bits.  All pages but the last are one."""
    length, page, heads, dim = 1_200_000_017, 65536, 16, 64
    cache, table = a_cache([2 * page], 1, dim, page, spare=0)
    table = table[:, :1].repeat(1, -(-length // page))
    table[:, -1] = 1 - table[0, 0]
    q, mask = normal(3, heads, dim, seed=66), torch.tensor([[1, 0, 0], [0, 1, 0], [1, 0, 1]], dtype=torch.uint8, device='cuda')
    own = table[0, -1].long() * page + torch.arange(length - 3, length, device='cuda') % page
    loud = torch.zeros((3, 1, dim), device='cuda')
    loud[:, 0, 0] = 400.0
    hidet_b200.quantized_cache_append(cache, loud, normal(3, 1, dim, seed=67, dtype=torch.float32), own)  # the drafted positions decide a row's result
    q[:, :, 0] = 8.0
    starts, n = ints(0, 3), ints(length)
    got = [attention_into(torch.empty_like(q), torch.empty(q.shape[:2], device='cuda'), q, cache, table, n, starts, mask, width) for width in (3, 1 << 30)]
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    v = hidet_b200.quantized_cache_read(cache, own, torch.float32)[1][:, 0]
    want = torch.stack([v[0], v[1], (v[0] + v[2]) / 2])[:, None].expand(3, heads, dim)
    assert (got[1][0].float() - want).abs().max() < 1e-2  # every other score is 300 below theirs


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [700, 32002, 200000])
@pytest.mark.parametrize('repeat', [1, 70])
def test_log_probs_of_rows_up_to_the_largest_number(dtype, vocab, repeat):
    """A token that is forced by the type's largest number has all the probability, and the entropy is zero; with two of them it is log 2."""
    most = torch.finfo(dtype).max
    x = normal(6, vocab, seed=68, dtype=torch.float32, std=3.0).to(dtype)
    x[0, vocab // 2] = most
    x[1, [3, vocab - 1]] = most
    x[2, 5] = most
    x[2, 6:9] = torch.tensor([0.72, 0.5, 0.3], dtype=torch.float64, device='cuda').mul(most).to(dtype)
    x[3] = -math.inf
    x[3, [0, vocab - 2]] = most
    x[4] = most
    x[5, 1] = 0.6 * most
    tokens = torch.full((6, 2), vocab - 1, device='cuda')
    tokens[:, 1] = 5
    for top in (0, 3, 32):
        got = check_log_probs(x.repeat(repeat, 1), tokens.repeat(repeat, 1), top)
        for at in range(0, 6 * repeat, 6):
            entropy = got[1][at:at + 6].tolist()
            # what is not at the largest number adds nothing: 16 bits hold it 16 apart from its neighbour
            assert entropy[0] == entropy[2] == entropy[5] == 0.0 and entropy[1] == pytest.approx(math.log(2.0), abs=1e-6) and entropy[3] == pytest.approx(math.log(2.0), abs=1e-6)
            assert entropy[4] == pytest.approx(math.log(vocab), abs=1e-5)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('heads,kv_heads,dim,tokens,long', FORMS[1:] + [(8, 2, 256, (3, 2), False)])
@pytest.mark.parametrize('size', [1e3, 1e9, 1e20])
@pytest.mark.parametrize('masked', [False, True])
def test_large_values_that_a_row_does_not_see_do_not_matter(dtype, heads, kv_heads, dim, tokens, long, size, masked):
    """The last token's value is larger than the others'.  It alone sees it; its neighbours' results stay, to the bit."""
    lengths = [700, 41]
    cache, table = a_cache(lengths, kv_heads, dim, 16)
    if long:
        cache, table = wide((cache, table))
    q, starts, n = normal(sum(tokens), heads, dim, seed=69, dtype=dtype), ints(0, tokens[0], sum(tokens)), ints(*lengths)
    mask = torch.zeros((sum(tokens), max(tokens)), dtype=torch.bool, device='cuda')
    for b, t in enumerate(tokens):
        mask[sum(tokens[:b]):sum(tokens[:b + 1]), :t] = torch.tril(torch.ones((t, t), dtype=torch.bool, device='cuda'))
    mask = mask if masked else None
    want = hidet_b200.quantized_cache_attention(q, cache, table, n, starts=starts, mask=mask, return_lse=True)
    for b, t in enumerate(tokens):
        last = slots_in(table, b, lengths[b], 16)[-1:]
        k, v = hidet_b200.quantized_cache_read(cache, last, torch.float32)
        hidet_b200.quantized_cache_append(cache, k, v * size, last)
    got = hidet_b200.quantized_cache_attention(q, cache, table, n, starts=starts, mask=mask, return_lse=True)
    first = 0
    for t in tokens:
        rows = slice(first, first + t - 1)
        assert torch.equal(got[0][rows], want[0][rows]) and torch.equal(got[1][rows], want[1][rows])
        first += t
    if size < 1e4 or dtype == torch.bfloat16:  # else the last token's results are beyond the type
        check_attention(lengths, list(tokens), heads, kv_heads, dim, 16, dtype, mask=mask, cache=(cache, table), q=q)


@pytest.mark.parametrize('heads,kv_heads,dim,tokens,long', FORMS)
def test_the_workspace_is_shared_with_the_linears(heads, kv_heads, dim, tokens, long):
    """Attention in many pieces and linears that meet in the workspace take turns at it, and its counters are zero in between."""
    lengths = [30000, 9000]
    cache, table = a_cache(lengths, kv_heads, dim, 64)
    if long:
        cache, table = wide((cache, table))
    q, starts, n = normal(sum(tokens), heads, dim, seed=70), ints(0, tokens[0], sum(tokens)), ints(*lengths)
    a, w = normal(2, 65536, seed=71), torch.randint(-128, 128, (65536, 128), dtype=torch.int8, device='cuda', generator=torch.Generator('cuda').manual_seed(72))
    scale = torch.full((128,), 1e-4, dtype=torch.float16, device='cuda')
    stream = torch.cuda.current_stream().cuda_stream
    first = None
    for _ in range(3):
        got = [hidet_b200.quantized_cache_attention(q, cache, table, n, starts=starts)]
        buffer = workspaces._buffers[(torch.cuda.current_device(), stream)]
        assert not buffer[:65536 * 4].any() and buffer[65536 * 4:].any()
        got.append(hidet_b200.symmetric_quant_matmul(a, w, scale))
        assert not workspaces._buffers[(torch.cuda.current_device(), stream)][:65536 * 4].any()
        first = first or got
        assert all(torch.equal(x, y) for x, y in zip(first, got))
    want = (a.double() @ w.double()) * scale.double()
    assert (first[1].double() - want).abs().max() <= (2.0 ** -11 + 2.0 ** -14) * want.abs().max()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [6000, 28772])
@pytest.mark.parametrize('repeat', [1, 30])
def test_log_probs_when_few_of_the_threads_have_all_the_large_ones(dtype, vocab, repeat):
    """Lists that overflow by vectors, by elements and not at all, of parts with 256 threads that take 16 bytes each in turn."""
    each, threads = 16 // dtype.itemsize, [0, 1, 16, 20, 40, 80, 200]
    at = torch.arange(vocab, device='cuda')
    rows = torch.stack([normal(vocab, seed=73 + i, dtype=torch.float32) + 60.0 * ((at // each) % 256 < n) for i, n in enumerate(threads)]).to(dtype)
    tokens = torch.arange(len(threads), device='cuda')
    for top in (1, 32):
        check_log_probs(rows.repeat(repeat, 1), tokens.repeat(repeat), top)


def test_rotary_into_elements_that_share_their_memory_is_refused():
    table, at = hidet_b200.rotary_table(16, 64), torch.arange(3, device='cuda')
    q = normal(3, 2, 64, seed=80)
    for out in (torch.empty_like(q)[:1].expand(3, 2, 64), torch.empty_like(q)[:, :1].expand(3, 2, 64)):
        with pytest.raises(ValueError, match='share'):
            hidet_b200.rotary_embedding(q, None, at, table, out=(out, None))
    whole = torch.empty((5, 2, 64), dtype=q.dtype, device='cuda')
    got = hidet_b200.rotary_embedding(q[:1], None, at[:1], table, out=(whole[:1, :1].expand(1, 1, 64).expand(1, 2, 64)[:, :1].as_strided((1, 2, 64), (0, 64, 1)), None))
    assert torch.equal(got[0], hidet_b200.rotary_embedding(q[:1], None, at[:1], table)[0])  # one token: its stride does not matter


@pytest.mark.parametrize('heads,kv_heads,dim,tokens,long', FORMS)
@pytest.mark.parametrize('q_std,k_std,scale', [(1e-28, 1.0, 1e27), (1e-36, 1.0, 1e29), (1e-37, 1e30, 1e6), (1e36, 1e-3, 1e-20), (1e-38, 1e-3, 1e-20), (1e20, 1e15, 1e-20)])
def test_queries_and_scales_of_any_size(heads, kv_heads, dim, tokens, long, q_std, k_std, scale):
    """A row's scores may be of ordinary size although its elements are not."""
    lengths = [700, 90]
    cache, table = a_cache(lengths, kv_heads, dim, 16)
    for b, n in enumerate(lengths):
        k, v = (normal(n, kv_heads, dim, seed=81 + i, dtype=torch.float32) for i in range(2))
        hidet_b200.quantized_cache_append(cache, k * k_std, v, slots_in(table, b, n, 16))
    if long:
        cache, table = wide((cache, table))
    q = (normal(sum(tokens), heads, dim, seed=83, dtype=torch.float32).double() * q_std).bfloat16()
    check_attention(lengths, list(tokens), heads, kv_heads, dim, 16, torch.bfloat16, cache=(cache, table), q=q, scale=scale)


@pytest.mark.parametrize('dtype,vocab', [(torch.float32, 409600), (torch.bfloat16, 819200), (torch.float16, 819193)])
def test_log_probs_of_the_longest_rows(dtype, vocab):
    logits = normal(3, vocab + 1, seed=90, dtype=dtype, std=3.0)
    check_log_probs(logits[:, :vocab], torch.tensor([0, vocab - 1, 77], device='cuda'), 20)
    if vocab * dtype.itemsize == 1638400:
        with pytest.raises(ffi.BackendException, match='are supported'):
            hidet_b200.token_log_probs(logits, torch.zeros(3, dtype=torch.int64, device='cuda'))
