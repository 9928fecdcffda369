"""GPU tests of the router's gradient where a score is close to 1 and the gradient a small difference of large terms.

Bounds (derived, elementwise), with u the half unit of the output type (its rounding, and fp32's before it for 16 bits) and
p, s the scores: everything before that rounding is 64-bit, with k products, E / 64 + 6 sums and one exponential of a unit or
two each, so the difference dw - mean is off by less than 2^-47 sum |dw|, times the score or slope in front of it; a factor's own
error is below 2^-40 of the result.  The exact values take 1 - p as the sum of the other scores, so nothing cancels.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = (torch.bfloat16, torch.float16, torch.float32)
HALF_UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SMALL = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}


@pytest.fixture(autouse=True)
def _gpu_only():
    if not torch.cuda.is_available():
        pytest.skip("ROCm GPU unavailable")


def rounding(dtype):
    return HALF_UNIT[dtype] + (0.0 if dtype is torch.float32 else 2.0 ** -23) + 2.0 ** -40


def normal(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("experts", [8, 64, 300, 896])
@pytest.mark.parametrize("k", [1, 2, 7])
def test_dense_gradient_of_a_confident_router(k, experts, dtype):
    """One logit 5 to 25 above the rest, softmax weights as they are: p (1 - p) dw is far below p dw."""
    from kernels import route_topk, route_topk_backward

    tokens = 11
    x = normal(experts, tokens, experts)
    for t in range(tokens):
        x[t, (37 * t) % experts] = x[t].max() + 5 + 2 * t
    x, dw = x.to(dtype), normal(k, tokens, k)
    _, chosen = route_topk(x.cuda(), k, normalize=False)
    actual = route_topk_backward(dw.cuda(), x.cuda(), chosen, normalize=False)
    assert actual.dtype is dtype
    y, index, dw = x.double(), chosen.cpu().long(), dw.double()
    e = torch.exp(y - y.amax(dim=1, keepdim=True))
    p = e / e.sum(dim=1, keepdim=True)
    weight = torch.zeros_like(y).scatter_(1, index, dw)  # dw of the chosen, 0 elsewhere
    # d_i = p_i sum_{j != i} p_j (dw_i - dw_j)
    exact = torch.stack([p[:, i] * (p * (weight[:, i:i + 1] - weight)).sum(dim=1) for i in range(experts)], dim=1)
    bound = rounding(dtype) * exact.abs() + 2.0 ** -47 * p * dw.abs().sum(dim=1, keepdim=True) + SMALL[dtype]
    worst = ((actual.cpu().double() - exact).abs() - bound).max()
    assert worst <= 0, float(worst)
