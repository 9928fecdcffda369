"""GPU tests of the router's ties between 0.0 and -0.0, which are one number: the lowest index wins, whatever the sign.

Choices are exact, against a stable descending sort of the logits on the CPU (where logits rank, equal ones are equal
scores).
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.fixture(autouse=True)
def _gpu_only():
    if not torch.cuda.is_available():
        pytest.skip("ROCm GPU unavailable")


def first_largest(c, k):
    return (c + 0.0).sort(dim=1, descending=True, stable=True).indices[:, :k]


def definition(x, k, groups, top_groups):
    c = x.double()
    if groups > 1:
        parts = c.view(len(x), groups, -1)
        drop = torch.ones(len(x), groups, dtype=torch.bool)
        drop.scatter_(1, first_largest(parts.amax(dim=2), top_groups), False)
        c = parts.masked_fill(drop[..., None], -INF).reshape(c.shape)
    return first_largest(c, k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts", [64, 256, 896])
def test_zeros_of_both_signs_are_equal(experts, score, dtype):
    """Short lists, long ones and lists past any; groups that lanes hold whole and groups that they do not."""
    from kernels import route_topk

    generator = torch.Generator().manual_seed(experts)
    x = torch.zeros(9, experts)
    x[torch.rand(9, experts, generator=generator) < 0.5] = -0.0
    x[1::3, ::5] = -1.5
    x[2::3, 3::11] = 1.0
    x[0] = -0.0
    x[0, experts // 2:] = 0.0  # all of the negative zeros come first
    x = x.to(dtype)
    for k in (2, 12, 40):
        for groups, top in ((1, 1), (8, 6), (32, 24)):
            for normalize in (True, False):
                _, chosen = route_topk(x.cuda(), k, score=score, groups=groups, top_groups=top, normalize=normalize)
                expected = definition(x, k, groups, top)
                assert torch.equal(chosen.cpu().long(), expected), (k, groups, normalize)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_masked_logits_tie_in_index_order(dtype):
    """Logits times a 0 / 1 mask: a negative one leaves -0.0."""
    from kernels import route_topk

    generator = torch.Generator().manual_seed(5)
    x = torch.randn(40, 128, generator=generator).abs().neg() * (torch.rand(40, 128, generator=generator) < 0.4)
    x[::2] = torch.where(x[::2] == 0, x[::2].abs(), x[::2])
    x[1::2, ::3] = x[1::2, ::3] + 0.0
    x = x.to(dtype)
    _, chosen = route_topk(x.cuda(), 8)
    assert torch.equal(chosen.cpu().long(), first_largest(x.double(), 8))
