"""GPU tests of what the router's and the sort's documentation says of extreme scores, flat ones and long lists."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu_only():
    if not torch.cuda.is_available():
        pytest.skip("ROCm GPU unavailable")


def test_weights_of_scores_that_underflow():
    """A softmax's normalised weights are the chosen logits' own softmax, also where every chosen score underflows; of
    sigmoids whose 64-bit scores are all 0 they are 0."""
    from kernels import route_topk

    x = torch.full((1, 64), -300.0, device="cuda")
    x[0, 0], x[0, 2] = 500.0, -299.0
    bias = torch.zeros(64, device="cuda")
    bias[0] = -10.0
    weights, chosen = route_topk(x, 2, bias=bias)
    assert chosen.tolist() == [[1, 2]]  # all 64-bit scores but the first are 0: ties
    exact = torch.softmax(torch.tensor([-300.0, -299.0], dtype=torch.float64), 0).cuda()
    assert bool(((weights[0].double() - exact).abs() <= 2.0 ** -23 * exact).all())
    weights, _ = route_topk(x, 2, bias=bias, normalize=False)
    assert not weights.any()
    weights, chosen = route_topk(torch.full((1, 16), -800.0, device="cuda"), 3, score="sigmoid")
    assert chosen.tolist() == [[0, 1, 2]] and not weights.any()


def test_scores_rank_by_their_logits_without_a_bias_and_in_64_bits_with_one():
    """Sigmoids past 37 are all 1 in 64 bits: by themselves their logits rank them, biased scores tie.  The same of softmax
    scores that underflow."""
    from kernels import route_topk

    x = torch.full((2, 32), -5.0, device="cuda")
    x[:, 3], x[:, 20], x[:, 9] = 40.0, 60.0, 50.0
    zero = torch.zeros(32, device="cuda")
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        y = x.to(dtype)
        assert route_topk(y, 3, score="sigmoid")[1].tolist() == [[20, 9, 3]] * 2
        assert route_topk(y, 3, score="sigmoid", bias=zero)[1].tolist() == [[3, 9, 20]] * 2
        y = (x - 800).to(dtype)
        y[:, 1] = 200.0
        assert route_topk(y, 4)[1].tolist() == [[1, 20, 9, 3]] * 2
        assert route_topk(y, 4, bias=zero)[1].tolist() == [[1, 0, 2, 3]] * 2


@pytest.mark.parametrize("experts,groups", [(896, 1), (256, 8), (1024, 1)])
def test_flat_routers(experts, groups):
    """Softmax scores near 1 / E, as of a router that has not learnt yet: closer than fp32 tells apart, so 64 bits decide."""
    from kernels import route_topk

    x = torch.randn(500, experts, generator=torch.Generator().manual_seed(experts)) * 0.02
    bias = torch.zeros(experts)
    _, chosen = route_topk(x.cuda(), 8, bias=bias.cuda(), groups=groups, top_groups=max(1, groups // 2), group_best=2)
    s = torch.softmax(x.double(), dim=1)
    if groups > 1:
        parts = s.view(500, groups, -1)
        best = parts.sort(dim=2, descending=True).values[..., :2].sum(dim=2)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, :groups // 2]
        drop = torch.ones_like(best, dtype=torch.bool).scatter_(1, kept, False)
        s = parts.masked_fill(drop[..., None], -1.0).reshape(s.shape)
    assert torch.equal(chosen.cpu().long(), s.sort(dim=1, descending=True, stable=True).indices[:, :8])


@pytest.mark.parametrize("tokens,k,experts,count,first", [
    (16384, 8, 256, 256, 0), (70001, 1, 1024, 1024, 0), (65536, 1, 40, 40, 0), (40000, 3, 128, 32, 32), (9000, 30, 7, 3, 5),
    (200003, 6, 300, 300, 0), (70000, 2, 50, 9, 60)])
def test_long_sorts_match_a_stable_sort(tokens, k, experts, count, first):
    """More than 1024 entries a workgroup: several rounds of counting and placing."""
    from kernels import sort_by_expert

    generator = torch.Generator().manual_seed(tokens)
    chosen = torch.randint(0, experts, (tokens, k), generator=generator, dtype=torch.int32)
    chosen[tokens // 3:tokens // 2] = experts // 2  # an uneven part
    order = sort_by_expert(chosen.cuda(), count, first=first)
    flat = chosen.flatten().long() - first
    here = (flat >= 0) & (flat < count)
    key = torch.where(here, flat, count)
    slots = key.sort(stable=True).indices
    used = int(here.sum())
    places = torch.full_like(slots, -1)
    places[slots[:used]] = torch.arange(used)
    slots[used:] = -1
    assert torch.equal(order.offs.cpu().long(), torch.bincount(key, minlength=count + 1)[:count].cumsum(0))
    assert torch.equal(order.slots.cpu().long(), slots)
    assert torch.equal(order.places.cpu().long().flatten(), places)
