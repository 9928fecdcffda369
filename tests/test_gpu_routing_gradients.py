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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("normalize", [False, True])
def test_gradient_of_saturated_sigmoids(normalize, dtype):
    """Logits far to both sides of 0: the slope s (1 - s) is e^-|x| / (1 + e^-|x|)^2, of which 1 - s keeps no bits past 37."""
    from kernels import route_topk_backward

    x = torch.tensor([[-40.0, -30.0, -20.0, -8.0, 0.0, 8.0, 14.0, 18.0, 22.0, 26.0, 30.0, 34.0, 36.0, 38.0, 42.0, 60.0]])
    if dtype is torch.float16:
        x = x / 4  # gradients of e^-15 at most are within its range
    chosen = torch.stack([torch.roll(torch.arange(16), r)[:3] for r in range(16)]).int()  # each three in turn
    x, dw = x.expand(16, 16).contiguous().to(dtype), normal(3, 16, 3)
    how = dict(score="sigmoid", normalize=normalize, scale=2.5)
    actual = route_topk_backward(dw.cuda(), x.cuda(), chosen.cuda(), **how)
    y, index, dw = x.double(), chosen.long(), 2.5 * dw.double()
    z = torch.exp(-y.abs())
    slope, s = (z / (1 + z) ** 2).gather(1, index), torch.sigmoid(y).gather(1, index)
    if normalize:
        # (dw_i - sum_j s_j dw_j / S) / S = sum_j s_j (dw_i - dw_j) / S^2
        total = s.sum(dim=1, keepdim=True)
        d = slope * (s[:, None] * (dw[:, :, None] - dw[:, None])).sum(dim=2) / total ** 2
        extra = 2.0 ** -47 * slope * dw.abs().sum(dim=1, keepdim=True) / total
    else:
        d, extra = slope * dw, 0 * dw
    exact = torch.zeros_like(y).scatter_(1, index, d)
    bound = rounding(dtype) * exact.abs() + torch.zeros_like(y).scatter_(1, index, extra) + SMALL[dtype]
    worst = ((actual.cpu().double() - exact).abs() - bound).max()
    assert worst <= 0, float(worst)


def test_gradient_of_normalised_sigmoids_that_are_tiny():
    """Logits near -700, whose scores are 1e-304: their ratios' gradient, w_i (dw_i - sum_j w_j dw_j) as a softmax's, is of
    ordinary size.  The scores' own 64-bit rounding, 2^-40 of them at most, is the error before the last rounding."""
    from kernels import route_topk_backward

    x = torch.tensor([[-700.0, -701.0, -699.0, 3.0], [-300.0, -300.0, -302.0, 3.0], [-120.0, -121.0, -125.0, 3.0]])
    chosen = torch.tensor([[0, 1, 2]] * 3, dtype=torch.int32)
    dw = 1e8 * normal(2, 3, 3)  # over 1e-304 past the largest 64-bit number
    actual = route_topk_backward(dw.cuda(), x.cuda(), chosen.cuda(), score="sigmoid").cpu().double()
    w, dw = torch.softmax(x[:, :3].double(), dim=1), dw.double()
    exact = w * (dw - (w * dw).sum(dim=1, keepdim=True))
    bound = rounding(torch.float32) * exact.abs() + 2.0 ** -40 * w * dw.abs().sum(dim=1, keepdim=True)
    assert bool(((actual[:, :3] - exact).abs() <= bound).all()) and not actual[:, 3].any()
