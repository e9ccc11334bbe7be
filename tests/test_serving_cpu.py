"""What the decoding operators refuse before they touch a GPU, and what of them needs none."""
import ctypes
import math

import pytest
import torch

import hidet_b200
from hidet_b200 import ffi
from hidet_b200.ffi import BF16, F16, F32, Heads

AT = 4096  # an address that nothing is read from: every call here is refused, or has no tokens


def heads(address=AT, token=512, head=64):
    return ctypes.byref(Heads(address, token, head))


def rotary(q=heads(), k=None, positions=AT, table=AT, tokens=2, n=4, kv=0, dim=64, rotary_dim=64, rows=16, layout=0, type=F16, bytes=8):
    return ffi.func('b200q_rotary_embedding')(q, k, q, k, positions, table, tokens, n, kv, dim, rotary_dim, rows, layout, type, bytes, None)


def append(cache=AT, pages=4, page_size=16, k=heads(), v=heads(), q=None, out=None, slots=AT, positions=None, table=None, tokens=2, n=0, kv=2, dim=64, rotary_dim=0, rows=0,
           layout=0, type=F16, slot_bytes=8, bytes=8):
    return ffi.func('b200q_quantized_cache_append')(cache, pages, page_size, k, v, q, out, slots, positions, table, tokens, n, kv, dim, rotary_dim, rows, layout, type, slot_bytes, bytes, None)


def read(cache=AT, pages=4, page_size=16, slots=AT, k=AT, v=AT, tokens=2, kv=2, dim=64, type=F16, slot_bytes=8):
    return ffi.func('b200q_quantized_cache_read')(cache, pages, page_size, slots, k, v, tokens, kv, dim, type, slot_bytes, None)


def attention(q=heads(), out=AT, cache=AT, pages=4, page_size=16, table=AT, width=2, lengths=AT, starts=None, mask=None, mask_width=0, batch=2, tokens=2, n=4, kv=2, dim=64, scale=0.125,
              type=F16, workspace=AT, nbytes=1 << 30):
    return ffi.func('b200q_quantized_cache_attention')(q, out, None, cache, pages, page_size, table, width, width, lengths, starts, mask, mask_width, mask_width, batch, tokens, n, kv, dim,
                                                       scale, type, workspace, nbytes, None)


def log_probs(logits=AT, stride=100, tokens=AT, out=AT, entropy=AT, top_out=AT, index=AT, rows=2, vocab=100, given=1, top=3, type=F16, bytes=8):
    return ffi.func('b200q_token_log_probs')(logits, stride, tokens, out, entropy, top_out, index, rows, vocab, given, top, type, bytes, None)


REFUSALS = [
    (rotary, dict(tokens=-1), 'negative'), (rotary, dict(type=7), 'type'), (rotary, dict(bytes=2), 'int32 or int64'), (rotary, dict(rotary_dim=63), ': '), (rotary, dict(rotary_dim=66), ': '),
    (rotary, dict(layout=5), ': '), (rotary, dict(q=None), 'null'), (rotary, dict(positions=None), 'null'), (rotary, dict(n=70000), 'heads'), (rotary, dict(tokens=1 << 40), 'tokens'),
    (append, dict(tokens=-1), 'negative'), (append, dict(type=3), 'type'), (append, dict(slot_bytes=1), 'int32 or int64'), (append, dict(dim=80), '80'), (append, dict(page_size=24), '24'),
    (append, dict(page_size=1 << 20), 'pages'), (append, dict(kv=0), ': '), (append, dict(k=None), 'null'), (append, dict(cache=None), ': '), (append, dict(cache=AT + 8), '16'),
    (append, dict(positions=AT, table=AT, rotary_dim=24, rows=8), 'multiples of 16'), (append, dict(q=heads(), n=4), ': '), (append, dict(tokens=1 << 40), 'tokens'),
    (read, dict(tokens=-1), 'negative'), (read, dict(type=9), 'type'), (read, dict(slot_bytes=0), 'int32 or int64'), (read, dict(dim=32), '32'), (read, dict(page_size=0), 'pages'),
    (read, dict(k=None), 'null'), (read, dict(k=AT + 8), 'aligned'), (read, dict(tokens=1 << 40), 'tokens'),
    (attention, dict(tokens=-1), 'negative'), (attention, dict(type=F32), 'float16 and bfloat16'), (attention, dict(n=3), '3 heads'), (attention, dict(kv=0), 'heads'),
    (attention, dict(page_size=40), '40'), (attention, dict(dim=100), '100'), (attention, dict(scale=0.0), 'positive'), (attention, dict(scale=math.nan), 'positive'),
    (attention, dict(scale=math.inf), 'positive'), (attention, dict(scale=-1.0), 'positive'), (attention, dict(tokens=3), 'starts'), (attention, dict(q=None), 'null'),
    (attention, dict(lengths=None), 'null'), (attention, dict(table=None), 'null'), (attention, dict(pages=0), '0 pages'), (attention, dict(q=heads(AT + 2)), 'aligned'),
    (attention, dict(q=heads(token=300)), 'strides'), (attention, dict(out=AT + 4), 'aligned'), (attention, dict(workspace=None), 'workspace'), (attention, dict(nbytes=1000), 'workspace'),
    (attention, dict(workspace=AT + 8), 'workspace'), (attention, dict(batch=1 << 21, tokens=1 << 21), 'sequences'), (attention, dict(tokens=1 << 40), 'tokens'),
    (log_probs, dict(rows=-1), 'negative'), (log_probs, dict(type=4), 'type'), (log_probs, dict(bytes=3), 'int32 or int64'), (log_probs, dict(vocab=0), 'no tokens'),
    (log_probs, dict(top=33), '33'), (log_probs, dict(top=5, vocab=4), '5 alternatives'), (log_probs, dict(stride=50), 'apart'), (log_probs, dict(logits=None), 'null'),
    (log_probs, dict(tokens=None), 'null'), (log_probs, dict(index=None), 'null'), (log_probs, dict(vocab=1 << 24, stride=1 << 24), 'rows of'), (log_probs, dict(rows=1 << 33), 'rows')]


@pytest.mark.parametrize('call,arguments,match', REFUSALS, ids=['{}-{}'.format(c.__name__, '-'.join(a)) for c, a, _ in REFUSALS])
def test_refusals(call, arguments, match):
    with pytest.raises(ffi.BackendException, match=match) as e:
        call(**arguments)
    assert 'cuda' not in str(e.value)  # it was refused here, not by the runtime


def test_calls_without_tokens_do_nothing():
    for call in (rotary, append, read, attention):
        assert call(tokens=0) == ffi.OK
    assert log_probs(rows=0) == ffi.OK and attention(batch=0, tokens=0) == ffi.OK


def test_attention_workspace():
    need = ffi.func('b200q_quantized_cache_attention_workspace_bytes')
    assert need(0, 1, 4, 2, 64) == need(1, 0, 4, 2, 64) == need(1, 1, 4, 2, 80) == 0
    assert 0 < need(1, 1, 32, 8, 128) == need(64, 64, 32, 8, 128) < need(64, 64 * 64, 32, 8, 128) < 1 << 26  # by the kind of call, not by its lengths
    with pytest.raises(ffi.BackendException, match='workspace of {} bytes'.format(need(2, 2, 4, 2, 64))):
        attention(nbytes=need(2, 2, 4, 2, 64) - 1)


def test_cpu_tensors_are_rejected():
    x, at = torch.zeros((2, 4, 64), dtype=torch.float16), torch.zeros(2, dtype=torch.int64)
    cache = hidet_b200.quantized_cache(2, 4, 64, 16, device='cpu')
    table, pages = hidet_b200.rotary_table(4, 64, device='cpu'), torch.zeros((2, 1), dtype=torch.int32)
    for call in (lambda: hidet_b200.rotary_embedding(x, None, at, table), lambda: hidet_b200.quantized_cache_append(cache, x, x, at), lambda: hidet_b200.quantized_cache_read(cache, at),
                 lambda: hidet_b200.quantized_cache_attention(x, cache, pages, pages[:, 0]), lambda: hidet_b200.token_log_probs(x[0], at)):
        with pytest.raises(ffi.BackendException, match='CUDA devices only'):
            call()


@pytest.mark.parametrize('scaling,factor', [(None, 1.0), ('linear', 4.0), ('ntk', 2.0), ('yarn', 4.0)])
def test_rotary_tables_hold_cosines_and_sines(scaling, factor):
    kwargs = dict(scaling=scaling, factor=factor, original_positions=64) if scaling else {}
    table = hidet_b200.rotary_table(100, 32, device='cpu', **kwargs)
    assert table.shape == (100, 32) and table.dtype == torch.float32
    size = (table[:, :16].double() ** 2 + table[:, 16:].double() ** 2).sqrt()
    # yarn lengthens every pair by 0.1 ln(factor) + 1
    assert (size - (0.1 * math.log(factor) + 1 if scaling == 'yarn' else 1.0)).abs().max() < 1e-6
    assert (table[0, 16:] == 0).all()
