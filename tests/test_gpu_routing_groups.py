"""GPU tests of expert groups by the sum of their two best biased scores, where those are large and of opposite signs.

Choices are exact.  Group sums lie 1e-6 or more apart, and 64-bit scores of up to 1e5 are within 2^-36 (1.5e-11), so the
64-bit definition's order does not hang on a rounding.
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


@pytest.mark.parametrize("experts,groups", [(64, 8), (256, 8), (256, 16), (896, 8), (120, 5)])
@pytest.mark.parametrize("size", [1e2, 1e3, 1e5])
@pytest.mark.parametrize("step", [5e-6, 5e-5, 5e-4])
def test_group_sums_of_large_terms_that_cancel(step, size, experts, groups):
    """Bias +B on the first of each group and -B on the rest: the sum of the two best is (s + B) + (s' - B), its fp32 terms off
    by up to 2^-24 B each.  s + s' is 0.9 and a multiple of ``step``, within 2^-23 for the logits' rounding."""
    from kernels import route_topk

    tokens, each = 50, experts // groups
    generator = torch.Generator().manual_seed(groups)
    s = torch.full((tokens, groups, each), 0.01, dtype=torch.float64)
    s[:, :, 0] = 0.55 + 0.2 * torch.rand(tokens, groups, generator=generator, dtype=torch.float64)
    for t in range(tokens):
        s[t, :, 1] = 0.9 + step * torch.randperm(groups, generator=generator) - s[t, :, 0]
    x = torch.logit(s).float()
    bias = torch.full((groups, each), -size)
    bias[:, 0] = size
    c = torch.sigmoid(x.double()) + bias.double()
    sums = c.sort(dim=2, descending=True).values[..., :2].sum(dim=2)
    for top in (groups // 2, 1):
        _, chosen = route_topk(x.view(tokens, experts).cuda(), top, score="sigmoid", bias=bias.flatten().cuda(),
                               groups=groups, top_groups=top, group_best=2)
        kept = sums.sort(dim=1, descending=True).indices[:, :top]
        # Of the kept groups the first experts, whose scores are the only ones above 0.
        first = c[:, :, 0].gather(1, kept)
        expected = kept.gather(1, first.sort(dim=1, descending=True).indices) * each
        assert torch.equal(chosen.cpu().long(), expected), top


@pytest.mark.parametrize("experts,groups", [(32, 4), (256, 8), (896, 8), (40, 5)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_a_group_sum_that_is_no_number_ranks_last(score, experts, groups):
    """A bias of inf beside -inf throughout a group: inf - inf, which no other group's sum is below."""
    from kernels import route_topk

    each = experts // groups
    x = torch.randn(20, experts, generator=torch.Generator().manual_seed(experts))
    bias = torch.zeros(experts)
    bias[:each] = -INF
    bias[1] = INF
    for top in (1, groups - 1):
        _, chosen = route_topk(x.cuda(), 2, score=score, bias=bias.cuda(), groups=groups, top_groups=top, group_best=2)
        assert int(chosen.min()) >= each and (chosen[:, 0] != chosen[:, 1]).all()
    _, chosen = route_topk(x.cuda(), 2, score=score, bias=bias.cuda(), groups=groups, group_best=2)
    assert (chosen[:, 0] == 1).all()  # all groups kept: the largest score
