"""Forward-mode derivatives, which no operator here has, are refused and not dropped: on the CPU, before any other check."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from kernels import (
    ExpertOrder,
    combine_rows,
    gather_rows,
    grouped_mm_mxfp4,
    grouped_mm_mxfp4_swiglu,
    matmul_mxfp4,
    route_topk,
)

W, S = torch.zeros(2, 8, 32, dtype=torch.uint8), torch.zeros(2, 8, 2, dtype=torch.uint8)
OFFS = torch.zeros(2, dtype=torch.int32)
ORDER = ExpertOrder(OFFS, torch.zeros(6, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32))
PRODUCTS = [lambda a: matmul_mxfp4(a, W[0], S[0]), lambda a: grouped_mm_mxfp4(a, W, S, OFFS),
            lambda a: grouped_mm_mxfp4_swiglu(a, W, S, OFFS)]
OTHERS = [lambda a: route_topk(a, 2), lambda a: gather_rows(a, ORDER), lambda a: combine_rows(a, ORDER),
          lambda a: combine_rows(torch.zeros(6, 4), ORDER, a)]


@pytest.mark.parametrize("call", PRODUCTS + OTHERS)
def test_forward_mode_is_refused(call):
    a = torch.zeros(3, 64)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            call(forward_ad.make_dual(a, torch.ones(3, 64)))
        with pytest.raises(ValueError, match="GPU|device|weights"):  # a tensor without a tangent: the next check
            call(a)


@pytest.mark.gpu
def test_differentiable_calls_beside_a_dual_level():
    """Tensors without a tangent run, and their gradients come, while another's forward-mode derivative is taken."""
    if not torch.cuda.is_available():
        pytest.skip("ROCm GPU unavailable")
    logits = torch.randn(5, 8, device="cuda").requires_grad_()
    with forward_ad.dual_level():
        weights, chosen = route_topk(logits, 2)
        weights[:, 0].sum().backward()
    assert logits.grad.abs().sum() > 0
    with torch.no_grad():
        assert torch.equal(route_topk(logits, 2)[0], weights)
