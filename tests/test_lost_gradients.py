"""4-bit products, which have no gradient, refuse rows that ask for one: on the CPU, before any other check."""

from __future__ import annotations

import pytest
import torch

from kernels import grouped_mm_mxfp4, grouped_mm_mxfp4_swiglu, matmul_mxfp4

W, S = torch.zeros(2, 8, 32, dtype=torch.uint8), torch.zeros(2, 8, 2, dtype=torch.uint8)
OFFS = torch.zeros(2, dtype=torch.int32)
PRODUCTS = [lambda a: matmul_mxfp4(a, W[0], S[0]), lambda a: grouped_mm_mxfp4(a, W, S, OFFS),
            lambda a: grouped_mm_mxfp4_swiglu(a, W, S, OFFS)]


@pytest.mark.parametrize("product", PRODUCTS)
def test_products_refuse_rows_that_ask_for_a_gradient(product):
    a = torch.zeros(3, 64, requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        product(a)
    with pytest.raises(ValueError, match="no gradient"):
        product(a * 2)
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):  # the next check
        product(a)
    with pytest.raises(ValueError, match="GPU"):
        product(a.detach())
