"""Logits of route_tokens as sums of floats: products of one sign, whose sums only grow, so that whatever cuts them instead of rounding adds up."""
import pytest
import torch

import hidet_b200

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('tokens,width', [(1, 4096), (9, 7168), (40, 16384)])
@pytest.mark.parametrize('count', [2, 16, 300])
def test_sums_of_one_sign(dtype, tokens, width, count):
    gen = torch.Generator(device='cuda').manual_seed(width + count)
    x = torch.rand(tokens, width, device='cuda', generator=gen).add_(0.5).to(dtype)
    x[:, 0] = 1.0
    router = torch.zeros(count, width, device='cuda', dtype=dtype)
    router[:-1] = (torch.rand(count - 1, width, device='cuda', generator=gen).add_(0.5) * (8.0 / width)).to(dtype)
    router[-1, 0] = 8.0     # an exact logit beside them
    chosen, weights = hidet_b200.route_tokens(x, router, 2 if count == 2 else 32 if count > 32 else count, normalize=False)
    logits = x.double() @ router.double().t()
    want = torch.softmax(logits, -1).gather(1, chosen.long())
    # A logit of up to 9 or so: eight sums of an instruction cut by a unit of 2^-23 (two for the sixteen products within), one rounding for every 256 of the width and ten for the rest.  It stands in
    # an exponent, whose own error and the quotient's are a few units; the share's denominator is off by as much again.
    off = float(logits.abs().max()) * (8 * 2 + width / 256 / 2 + 10) * 2.0 ** -23
    assert torch.all((weights.double() - want).abs() <= want * (2 * off + 12 * 2.0 ** -23))
