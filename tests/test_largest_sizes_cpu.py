"""Sizes whose last steps 32-bit indices of the kernels would not hold are refused before anything is launched."""
import pytest

from hidet_b200 import ffi
from test_tokens_experts_cpu import product, tokens


# a CTA's threads take eight elements each and step by 8192: the step behind the last element has to be a number too
@pytest.mark.parametrize('width', [2 ** 31 - 8191, 0x7fffff00, 2 ** 31])
@pytest.mark.parametrize('norm', [None, 4096])
def test_tokens_too_wide_for_a_step(width, norm):
    with pytest.raises(ffi.BackendException, match='elements'):
        tokens(width=width, stride=width, norm=norm)


# tiles have up to 256 rows or columns
@pytest.mark.parametrize('size', [2 ** 31 - 255, 2 ** 31 - 1])
@pytest.mark.parametrize('layout', [0, 1])
@pytest.mark.parametrize('k', [1, 16])
def test_products_too_large_for_a_tile(size, layout, k):
    for sizes in (dict(m=size, n=16), dict(m=1, n=size)):
        with pytest.raises(ffi.BackendException, match='2\\^31'):
            product(k=k, layout=layout, **sizes)
