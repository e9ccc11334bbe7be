"""quantize_tokens behind a norm of rows so small that their squares are no numbers of float, with an eps of nothing or next to it: a row's size then cancels."""
import pytest
import torch

import hidet_b200
import token_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('width', [64, 200, 1000, 4096, 4100, 20000, 40002])
@pytest.mark.parametrize('eps', [0.0, 1e-42, 1e-36])
def test_tiny_rows(width, dtype, eps):
    gen = torch.Generator(device='cuda').manual_seed(width)
    size = torch.tensor([2.0 ** -e for e in (0, 30, 48, 52, 60, 70, 75, 80, 90)], device='cuda', dtype=torch.float64)[:, None]
    x = (torch.randn(9, width, device='cuda', generator=gen).double() * size).to(dtype)
    norm = (1 + 0.2 * torch.randn(width, device='cuda', generator=gen)).to(dtype)
    codes, scales = hidet_b200.quantize_tokens(x, norm, eps)
    exact, want = ref.quantized(x, norm, float(torch.tensor(eps, dtype=torch.float32)))
    assert (codes.double() - exact).abs().max() <= 0.5 + 127 * 4 * 2.0 ** -24
    # as for rows of ordinary size: a sum of squares in parts of at most 64 elements a thread (40 with the longest row here) and 10 additions, a quotient, a sum, a root, two quotients; and a square
    # below 2^-126 is off by 2^-150 at most, which is 2^-50 of a mean of 2^-100
    n = 8 + (64 + 16) / 2
    assert torch.all((scales.double() - want).abs() <= want * n * 2.0 ** -24)
