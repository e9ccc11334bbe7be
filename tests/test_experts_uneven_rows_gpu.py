"""Layers of experts over rows whose elements differ much in size: x and h are held against their row's largest element, and no worse than the documentation says."""
import pytest
import torch

import hidet_b200
import token_reference
from hidet_b200 import ffi

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def rows(gen, tokens, hidden, dtype, kind):
    x = torch.randn(tokens, hidden, device='cuda', generator=gen)
    if kind == 'ramp':      # every size from the largest down to 2^-24 of it
        x = torch.sign(x) * torch.exp2(-24 * torch.rand(tokens, hidden, device='cuda', generator=gen))
    else:                   # two channels far larger than the others, by 2^kind
        x[:, [3, hidden // 2 + 1]] = torch.sign(x[:, [3, hidden // 2 + 1]]) * 2.0 ** kind
    return x.to(dtype)


# few tokens, several an expert, many, and the kernels for any alignment
@pytest.mark.parametrize('tokens,hidden,inner,count,top', [(1, 512, 256, 8, 2), (19, 1024, 512, 8, 2), (200, 512, 256, 8, 2), (5, 136, 40, 4, 2)])
@pytest.mark.parametrize('dtype,kind', [(F16, 6), (F16, 12), (F16, 'ramp'), (BF16, 6), (BF16, 14), (BF16, 24), (BF16, 'ramp')])
@pytest.mark.parametrize('blind', [False, True])
def test_rows_of_unlike_elements(tokens, hidden, inner, count, top, dtype, kind, blind):
    """blind: the weights have zeros where the tokens are large, so that nothing hides how the others are held; h is uneven too, its scales lie between 2^-10 and 1."""
    gen = torch.Generator(device='cuda').manual_seed(tokens + hidden)
    x = rows(gen, tokens, hidden, dtype, kind)
    gate_up, down = (torch.randint(-127, 128, shape, device='cuda', generator=gen, dtype=torch.int8) for shape in ((count, 2 * inner, hidden), (count, hidden, inner)))
    if blind:
        gate_up[:, :, [3, hidden // 2 + 1]] = 0
    s1 = torch.exp2(-10 * torch.rand(count, 2 * inner, device='cuda', generator=gen)) / (64 * hidden ** 0.5)
    if not blind and kind != 'ramp':
        s1 = s1 * 2.0 ** -kind
    s2 = torch.rand(count, hidden, device='cuda', generator=gen) / (64 * inner ** 0.5)
    chosen = torch.randint(0, count, (tokens, top), device='cuda', generator=gen, dtype=torch.int32)
    weights = torch.rand(tokens, top, device='cuda', generator=gen)
    got = hidet_b200.mixture_of_experts(x, chosen, weights, gate_up, s1, down, s2)
    want, bound = token_reference.experts(x, chosen, weights, gate_up, s1, down, s2, None)
    token_reference.check(got, want, bound)
    assert torch.equal(got, hidet_b200.mixture_of_experts(x, chosen, weights, gate_up, s1, down, s2))
    assert ffi.func('b200q_check_status')() == ffi.OK
