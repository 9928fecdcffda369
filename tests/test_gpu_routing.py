"""GPU tests of the router, the sort by expert and the way to sorted rows and back, against their definitions in 64 bits.

Bounds (derived, elementwise), with u the half unit of the output type:

* choices are exact: scores are compared in 64 bits, and logits whose 64-bit scores tie by rounding are not drawn;
* weights: 2^-24 of their size for the rounding to fp32, and 2^-40 for the 64-bit arithmetic before it;
* the logits' gradient: u of its size, and 2^-22 of its two terms' sizes where they are added in fp32;
* combine: each of k products and sums rounds once, (k + 2) 2^-23 sum |w y|, and u of the result;
* dy: one fp32 product and one rounding, (u + 2^-23) |w dout|; dw: (H / 64 + 16) 2^-23 sum |dout y|, since a lane
  adds H / 64 products and the 64 lanes meet in 6 steps.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = (torch.bfloat16, torch.float16, torch.float32)
HALF_UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SMALL = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}
INF = float("inf")


@pytest.fixture(autouse=True)
def _gpu_only():
    if not torch.cuda.is_available():
        pytest.skip("ROCm GPU unavailable")


def normal(seed, *shape):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def within(actual, exact, bound):
    worst = float(((actual.double() - exact).abs() - bound).max()) if actual.numel() else -1.0
    assert worst <= 0, worst


def first_largest(scores, k):
    """Indices of the k largest of each row, ties to the lowest index."""
    return scores.sort(dim=1, descending=True, stable=True).indices[:, :k]


def scores_of(x, score):
    x = x.double()
    if score == "sigmoid":
        return torch.sigmoid(x)
    e = torch.exp(x - x.amax(dim=1, keepdim=True))
    return e / e.sum(dim=1, keepdim=True)


def route(x, k, score, bias, groups, top_groups, group_best, normalize, scale):
    """The definition: (weights, experts)."""
    s = scores_of(x, score)
    c = s if bias is None else s + bias.double()
    if groups > 1:
        parts = c.view(len(x), groups, -1)
        best = parts.sort(dim=2, descending=True).values[..., :group_best].sum(dim=2)
        drop = torch.ones_like(best, dtype=torch.bool).scatter_(1, first_largest(best, top_groups), False)
        c = parts.masked_fill(drop[..., None], -INF).view_as(c)
    chosen = first_largest(c, k)
    w = s.gather(1, chosen)
    if normalize:
        w = w / w.sum(dim=1, keepdim=True)
    return w * scale, chosen


ROUTES = [
    # tokens, experts, k, score, bias, groups, top_groups, group_best, normalize, scale
    (1, 1, 1, "softmax", False, 1, 1, 1, True, 1.0),
    (1, 256, 8, "sigmoid", True, 8, 4, 2, True, 2.5),
    (5, 8, 2, "softmax", False, 1, 1, 1, True, 1.0),
    (67, 65, 7, "softmax", True, 5, 2, 2, False, 1.0),
    (130, 128, 8, "softmax", False, 1, 1, 1, True, 1.0),
    (33, 896, 16, "softmax", False, 1, 1, 1, False, 1.0),
    (33, 896, 16, "sigmoid", True, 1, 1, 1, True, 2.0),
    (40, 160, 6, "softmax", False, 8, 3, 1, False, 16.0),
    (19, 1024, 64, "sigmoid", True, 512, 200, 2, True, 1.0),
    (21, 1000, 33, "sigmoid", False, 1000, 40, 2, False, 1.0),
    (9, 64, 64, "sigmoid", False, 1, 1, 1, True, 1.0),
    (7, 96, 4, "sigmoid", False, 4, 1, 2, True, 1.0),
    (300, 24, 3, "softmax", True, 4, 2, 1, True, 1.0),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ROUTES)
def test_route_matches_the_definition(case, dtype):
    from kernels import route_topk

    tokens, experts, k, score, biased, groups, top, best, normalize, scale = case
    x = (normal(tokens + experts, tokens, experts) * 1.5).to(dtype)
    bias = normal(3, experts) * 0.3 if biased else None
    weights, chosen = route_topk(x, k, score=score, bias=bias, groups=groups, top_groups=top, group_best=best,
                                 normalize=normalize, scale=scale)
    expected, indices = route(x, k, score, bias, groups, top, best, normalize, scale)
    assert weights.dtype is torch.float32 and chosen.dtype is torch.int32
    assert torch.equal(chosen.long(), indices)
    within(weights, expected, (2.0 ** -24 + 2.0 ** -40) * expected.abs() + 2.0 ** -149)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_equal_scores_go_to_the_lowest_index(score):
    from kernels import route_topk

    x = torch.zeros(3, 130, device="cuda")
    x[1] = (torch.arange(130, device="cuda") // 3 % 5).float()
    x[2, ::7] = 2.0
    for bias in (None, torch.zeros(130, device="cuda")):
        for groups, top in ((1, 1), (10, 4)):
            _, chosen = route_topk(x, 9, score=score, bias=bias, groups=groups, top_groups=top)
            _, expected = route(x, 9, score, bias, groups, top, 1, True, 1.0)
            assert torch.equal(chosen.long(), expected)


def test_close_scores_are_told_apart():
    """Logits one fp32 step apart, and scores that differ by a bias of 2^-40: fp32 scores would tie."""
    from kernels import route_topk

    one = torch.tensor(1.0)
    x = torch.full((2, 64), 1.0, device="cuda")
    x[:, 40] = torch.nextafter(one, one + 1).item()
    bias = torch.zeros(64, device="cuda")
    bias[50] = 2.0 ** -40
    for score in ("softmax", "sigmoid"):
        assert route_topk(x, 1, score=score)[1].flatten().tolist() == [40, 40]
        assert route_topk(torch.ones(1, 64, device="cuda"), 2, score=score, bias=bias)[1].flatten().tolist() == [50, 0]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [True, False])
def test_masked_logits(score, normalize):
    """-inf logits: experts that cannot be told apart come in index order with weight 0; a row of them has weights 0."""
    from kernels import route_topk, route_topk_backward

    x = normal(5, 4, 70)
    x[0] = -INF
    x[1, 3:] = -INF
    x[2, ::2] = -INF
    x[3, :] = torch.finfo(torch.float32).min
    weights, chosen = route_topk(x, 5, score=score, normalize=normalize)
    assert chosen[0].tolist() == [0, 1, 2, 3, 4] and not weights[0].any()
    assert set(chosen[1, :3].tolist()) == {0, 1, 2} and chosen[1, 3:].tolist() == [3, 4]
    assert not weights[1, 3:].any() and (weights[1, :3] > 0).all()
    expected, indices = route(x[2:3], 5, score, None, 1, 1, 1, normalize, 1.0)
    assert torch.equal(chosen[2:3].long(), indices)
    within(weights[2:3], expected, 2.0 ** -23 * expected)
    assert torch.isfinite(weights).all()
    dx = route_topk_backward(torch.ones(4, 5, device="cuda"), x, chosen, score=score, normalize=normalize)
    assert torch.isfinite(dx).all() and not dx[0].any() and not dx[x == -INF].any()


def test_nan_and_infinite_logits_keep_choices_valid():
    from kernels import route_topk

    x = normal(8, 4, 100)
    x[0, 17] = float("nan")
    x[1] = float("nan")
    x[2, 60] = INF
    weights, chosen = route_topk(x, 6)
    assert torch.isnan(weights[:2]).all() and 17 not in chosen[0].tolist()
    assert chosen[1].tolist() == list(range(6)) and chosen[2, 0] == 60
    weights, chosen = route_topk(x, 6, score="sigmoid")
    assert torch.isfinite(weights[0]).all() and 17 not in chosen[0].tolist() and torch.isnan(weights[1]).all()
    assert chosen[2, 0] == 60 and torch.isfinite(weights[2]).all()
    for each in (chosen, route_topk(x, 6, bias=torch.full((100,), -INF, device="cuda"))[1]):
        assert ((each >= 0) & (each < 100)).all() and all(len(set(r)) == 6 for r in each.tolist())


def test_scores_that_are_no_numbers_keep_choices_valid():
    """inf - inf and NaN made by the bias, over few experts and many: distinct indices, whatever their order."""
    from kernels import route_topk

    for experts in (8, 16, 200, 896):
        x = normal(experts, 3, experts)
        x[1, 5] = INF
        for bad in (-INF, INF, float("nan")):
            for score in ("softmax", "sigmoid"):
                _, chosen = route_topk(x, 4, score=score, bias=torch.full((experts,), bad, device="cuda"))
                assert ((chosen >= 0) & (chosen < experts)).all() and all(len(set(r)) == 4 for r in chosen.tolist())


def test_many_equal_and_nearly_equal_scores():
    """More ties at the k-th place than any short list holds, and scores one fp32 step apart throughout."""
    from kernels import route_topk

    step = 1 + torch.arange(256, device="cuda", dtype=torch.float64) * 2.0 ** -23
    rows = torch.stack([torch.zeros(256, device="cuda"), step.float(), step.flip(0).float(),
                        (torch.arange(256, device="cuda") % 3).float()])
    bias = torch.zeros(256, device="cuda")
    bias[::5] = 2.0 ** -30
    for score in ("softmax", "sigmoid"):
        for b in (None, bias):
            for groups, top, best in ((1, 1, 1), (8, 4, 2), (16, 5, 1)):
                _, chosen = route_topk(rows, 12, score=score, bias=b, groups=groups, top_groups=top, group_best=best)
                _, expected = route(rows, 12, score, b, groups, top, best, True, 1.0)
                assert torch.equal(chosen.long(), expected), (score, b is None, groups)


def test_extreme_scores_keep_their_ratios():
    """Normalised weights of logits that all underflow beside a larger, ineligible one."""
    from kernels import route_topk

    x = torch.full((1, 64), -300.0, device="cuda")
    x[0, 0] = 500.0
    x[0, 5] = -299.0
    bias = torch.zeros(64, device="cuda")
    bias[0] = -10.0
    weights, chosen = route_topk(x, 2, bias=bias)
    assert chosen.tolist() == [[5, 1]] or chosen.tolist() == [[1, 2]] or 0 not in chosen[0].tolist()
    assert abs(float(weights.sum()) - 1) < 2.0 ** -22
    weights, _ = route_topk(x[:, 1:].contiguous(), 2, score="sigmoid")
    exact = torch.softmax(torch.tensor([-299.0, -300.0], dtype=torch.float64), 0).cuda()
    within(weights[0], exact, 2.0 ** -23 * exact)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ROUTES)
def test_route_gradient(case, dtype):
    from kernels import route_topk, route_topk_backward

    tokens, experts, k, score, biased, groups, top, best, normalize, scale = case
    x = (normal(tokens + experts, tokens, experts) * 1.5).to(dtype)
    bias = normal(3, experts) * 0.3 if biased else None
    dw = normal(4, tokens, k)
    how = dict(score=score, normalize=normalize, scale=scale)
    _, chosen = route_topk(x, k, bias=bias, groups=groups, top_groups=top, group_best=best, **how)
    dx = route_topk_backward(dw, x, chosen, **how)
    y = x.double().requires_grad_()
    s = torch.sigmoid(y) if score == "sigmoid" else torch.softmax(y, dim=1)
    w = s.gather(1, chosen.long())
    if normalize:
        w = w / w.sum(dim=1, keepdim=True)
    (w * scale).backward(dw.double())
    size = scale * dw.double().abs().sum(dim=1, keepdim=True) * torch.ones_like(y)
    assert dx.dtype is dtype and dx.is_contiguous()
    within(dx, y.grad, HALF_UNIT[dtype] * (1 + 2.0 ** -10) * y.grad.abs() + 2.0 ** -22 * s.detach() * size
           + 2.0 ** -40 * size + SMALL[dtype])


def test_route_gradient_against_differences():
    """(f(x + h) - f(x - h)) / 2h of the loss, in fp32 weights rounded to 2^-24 each: their error over 2h = 2^-7 is below
    2^-24 * 4 * sum|dw| * 2^7, the differences' own h^2 / 6 times a third derivative of at most 2 * sum|dw|."""
    from kernels import route_topk

    for score in ("softmax", "sigmoid"):
        for normalize in (True, False):
            x = normal(11, 1, 12).requires_grad_()
            dw = normal(12, 1, 3)
            weights, chosen = route_topk(x, 3, score=score, normalize=normalize)
            (weights * dw).sum().backward()
            h, size = 2.0 ** -8, float(dw.abs().sum())
            for i in range(12):
                step = torch.zeros_like(x)
                step[0, i] = h
                with torch.no_grad():
                    up, above = route_topk(x + step, 3, score=score, normalize=normalize)
                    down, below = route_topk(x - step, 3, score=score, normalize=normalize)
                if not (torch.equal(above, chosen) and torch.equal(below, chosen)):
                    continue  # the choice changes there
                slope = float(((up - down) * dw).sum()) / (2 * h)
                assert abs(slope - float(x.grad[0, i])) <= (2.0 ** -15 + h * h) * size, (score, normalize, i)


def test_route_strides_and_empty_batches():
    from kernels import route_topk, route_topk_backward

    base = normal(2, 50, 300).to(torch.bfloat16)
    for view in (base[:, 3:131], base[::3, :70], base[7:8], base[:1].expand(6, 300)):
        weights, chosen = route_topk(view, 4)
        w0, c0 = route_topk(view.contiguous(), 4)
        assert torch.equal(weights, w0) and torch.equal(chosen, c0)
        dw = normal(1, *weights.shape)
        assert torch.equal(route_topk_backward(dw, view, chosen), route_topk_backward(dw, view.contiguous(), chosen))
    weights, chosen = route_topk(base[:0], 4)
    assert weights.shape == chosen.shape == (0, 4)
    assert route_topk_backward(weights, base[:0], chosen).shape == (0, 300)


def test_route_of_many_tokens():
    """More tokens than one launch has waves."""
    from kernels import route_topk, route_topk_backward

    tokens = (1 << 18) + 7
    x = normal(4, tokens, 8)
    weights, chosen = route_topk(x, 2)
    expected, indices = route(x, 2, "softmax", None, 1, 1, 1, True, 1.0)
    assert torch.equal(chosen.long(), indices)
    within(weights, expected, 2.0 ** -23 * expected)
    dx = route_topk_backward(torch.ones_like(weights), x, chosen)
    assert float(dx.abs().max()) < 2.0 ** -40  # the weights of a token sum to 1 whatever the logits


def sorted_reference(experts, count, first):
    flat = experts.flatten().cpu().tolist()
    lists = [[] for _ in range(count)]
    for slot, e in enumerate(flat):
        if first <= e < first + count:
            lists[e - first].append(slot)
    slots = sum(lists, [])
    offs = torch.tensor([len(part) for part in lists]).cumsum(0)
    places = torch.full((len(flat),), -1)
    places[torch.tensor(slots, dtype=torch.long)] = torch.arange(len(slots))
    return offs.int(), torch.tensor(slots + [-1] * (len(flat) - len(slots)), dtype=torch.int32), places.int()


@pytest.mark.parametrize("tokens,k,experts,count,first", [
    (1, 1, 1, 1, 0), (1, 8, 256, 256, 0), (5, 3, 7, 7, 0), (64, 8, 128, 128, 0), (100, 4, 128, 32, 32), (2049, 1, 3, 3, 0),
    (3000, 8, 1024, 1024, 0), (4096, 8, 256, 256, 0), (777, 16, 896, 224, 672), (20000, 2, 64, 64, 0), (300, 2, 5, 4, 3),
    (1, 5000, 40, 40, 0)])
def test_sort_matches_the_definition(tokens, k, experts, count, first):
    from kernels import sort_by_expert

    generator = torch.Generator(device="cuda").manual_seed(tokens + k)
    chosen = torch.randint(0, experts, (tokens, k), device="cuda", generator=generator, dtype=torch.int32)
    order = sort_by_expert(chosen, count, first=first)
    offs, slots, places = sorted_reference(chosen, count, first)
    assert torch.equal(order.offs.cpu(), offs) and torch.equal(order.slots.cpu(), slots)
    assert torch.equal(order.places.cpu().flatten(), places) and order.places.shape == (tokens, k)


def test_sort_of_one_expert_none_and_any_numbers():
    from kernels import sort_by_expert

    one = torch.full((700, 8), 5, device="cuda", dtype=torch.int32)
    order = sort_by_expert(one, 9)
    assert order.offs.tolist() == [0] * 5 + [5600] * 4 and torch.equal(order.slots, torch.arange(5600, device="cuda").int())
    order = sort_by_expert(one, 5)
    assert not order.offs.any() and (order.slots == -1).all() and (order.places == -1).all()
    order = sort_by_expert(one[:0], 5)
    assert order.offs.tolist() == [0] * 5 and order.slots.numel() == 0 and order.places.shape == (0, 8)
    odd = torch.tensor([[-1, 2 ** 31 - 1, -2 ** 31, 3, 1024, 0]], device="cuda", dtype=torch.int32)
    order = sort_by_expert(odd, 1024)
    assert order.places.tolist() == [[-1, -1, -1, 1, -1, 0]] and order.slots.tolist() == [5, 3, -1, -1, -1, -1]
    order = sort_by_expert(odd, 1, first=2 ** 31 - 1)
    assert order.places.tolist() == [[-1, 0, -1, -1, -1, -1]]


def order_of(seed, tokens, k, experts, count=None, first=0):
    from kernels import sort_by_expert

    generator = torch.Generator(device="cuda").manual_seed(seed)
    chosen = torch.rand(tokens, experts, device="cuda", generator=generator).topk(k, dim=1).indices.to(torch.int32)
    return sort_by_expert(chosen, count or experts, first=first)


def gathered(x, order, rows):
    out = torch.zeros(rows, x.shape[1], dtype=x.dtype, device=x.device)
    slots = order.slots[:rows].long()
    used = slots >= 0
    out[:len(slots)][used] = x[slots[used] // order.places.shape[1]]
    return out


def rows_of(y, order):
    """[T, k, H] in 64 bits: each slot's row, zeros where it has none."""
    places = order.places.long()
    here = (places >= 0) & (places < len(y))
    if len(y) == 0:
        return torch.zeros(*places.shape, y.shape[1], dtype=torch.float64, device=y.device)
    return y.double()[places.clamp(0, len(y) - 1)] * here[..., None]


ROWS = [
    # tokens, k, experts, local, first, H, room for rows (None: all)
    (1, 1, 1, 1, 0, 1, None), (1, 8, 256, 256, 0, 7168, None), (33, 4, 16, 16, 0, 2880, None), (64, 8, 128, 128, 0, 2048, None),
    (50, 6, 40, 10, 20, 333, None), (50, 6, 40, 10, 20, 264, 40), (17, 2, 8, 8, 0, 8, 100), (129, 16, 896, 224, 0, 72, 500),
    (5, 3, 9, 9, 0, 4097, 15), (3, 1, 4, 4, 0, 16, 0), (40, 20, 32, 32, 0, 136, None)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ROWS)
def test_rows_there_and_back(case, dtype):
    from kernels import combine_rows, combine_rows_backward, gather_rows

    tokens, k, experts, local, first, h, rows = case
    order = order_of(tokens, tokens, k, experts, local, first)
    x = normal(1, tokens, h).to(dtype)
    count = tokens * k if rows is None else rows
    xs = gather_rows(x, order, rows=rows)
    assert torch.equal(xs, gathered(x, order, count))
    y, w, dout = normal(2, count, h).to(dtype), normal(3, tokens, k), normal(4, tokens, h).to(dtype)
    if int(order.offs[-1]) < count:
        y[int(order.offs[-1]):] = float("nan")  # rows of no token are not read
    each = rows_of(torch.nan_to_num(y), order)
    for weights in (w, None):
        factor = torch.ones_like(w) if weights is None else w
        terms = each * factor.double()[..., None]
        out = combine_rows(y, order, weights)
        exact = terms.sum(dim=1)
        within(out, exact, HALF_UNIT[dtype] * exact.abs() + (k + 2) * 2.0 ** -23 * terms.abs().sum(dim=1) + SMALL[dtype])
        dy, dw = combine_rows_backward(dout, y, order, weights)
        scaled = torch.zeros(count, h, dtype=torch.float64, device="cuda")
        slots = order.slots[:count].long()
        used = slots >= 0
        scaled[:len(slots)][used] = dout.double()[slots[used] // k] * factor.double().flatten()[slots[used], None]
        within(dy, scaled, (HALF_UNIT[dtype] + 2.0 ** -23) * scaled.abs() + SMALL[dtype])
        products = dout.double()[:, None] * each
        within(dw, products.sum(dim=2), (h / 64 + 16) * 2.0 ** -23 * products.abs().sum(dim=2) + 2.0 ** -126)
        assert dy.dtype is dtype and dw.dtype is torch.float32
    only_dy, none = combine_rows_backward(dout, y, order, w, need_dweights=False)
    none_too, only_dw = combine_rows_backward(dout, y, order, w, need_dy=False)
    assert none is None and none_too is None
    dy, dw = combine_rows_backward(dout, y, order, w)
    assert torch.equal(only_dy, dy) and torch.equal(only_dw, dw)


def test_gather_of_other_types_strides_and_alignments():
    from kernels import combine_rows, combine_rows_backward, gather_rows, quantize_fp8

    order = order_of(9, 70, 3, 12)
    wide = normal(6, 70, 400)
    q, scale = quantize_fp8(wide)
    assert torch.equal(gather_rows(q, order).view(torch.uint8), gathered(q.view(torch.uint8), order, 210))
    scale = scale.contiguous()
    assert torch.equal(gather_rows(scale, order), gathered(scale, order, 210))
    for x in (wide.int(), wide.half()[:, 1:200], wide.to(torch.uint8)[:, 3:10], wide[:, 2:], wide.half()[:1].expand(70, 400)):
        assert torch.equal(gather_rows(x, order), gathered(x, order, 210))
    y = normal(7, 210, 402).to(torch.bfloat16)
    dout = normal(8, 70, 402).to(torch.bfloat16)
    for lo, hi in ((1, 400), (2, 10), (0, 401), (8, 400)):
        part, gradient = y[:, lo:hi], dout[:, lo:hi]
        assert torch.equal(combine_rows(part, order), combine_rows(part.contiguous(), order))
        dy, dw = combine_rows_backward(gradient, part, order)
        assert torch.equal(dy, combine_rows_backward(gradient.contiguous(), part.contiguous(), order)[0])
        # dw's order of products is that of the loads, whose width the alignment decides; any order of them is within the bound
        # at the head of this file, whose steps count products a lane and not which ones.
        products = gradient.double()[:, None] * rows_of(part, order)
        within(dw, products.sum(dim=2), ((hi - lo) / 64 + 16) * 2.0 ** -23 * products.abs().sum(dim=2))


def test_rows_past_four_gib():
    from kernels import combine_rows, combine_rows_backward, gather_rows

    tokens, k, h = 90000, 4, 8192
    order = order_of(3, tokens, k, 16)
    x = torch.empty(tokens, h, device="cuda", dtype=torch.bfloat16).normal_()
    xs = gather_rows(x, order)
    assert xs.numel() * 2 > 5 << 30
    for t in (0, tokens // 2, tokens - 1):
        assert torch.equal(xs[order.places[t].long()], x[t].expand(k, h))
    back = combine_rows(xs, order)
    assert torch.equal(back, x * 4)
    dy, dw = combine_rows_backward(x, xs, order)
    assert torch.equal(dy, xs)
    squares = x[-8:].double().square().sum(dim=1, keepdim=True)
    within(dw[-8:], squares.expand(8, k), (h / 64 + 16) * 2.0 ** -23 * squares)


def test_places_that_point_nowhere_are_skipped():
    from kernels import combine_rows, combine_rows_backward, gather_rows

    order = order_of(4, 20, 2, 6)
    bad = order.places.clone()
    bad[3, 0], bad[4, 1], bad[5] = 2 ** 31 - 1, -2 ** 31, -1
    order = order._replace(places=bad)
    y = normal(2, 40, 24)
    each = rows_of(y, order)
    within(combine_rows(y, order), each.sum(dim=1), 4 * 2.0 ** -23 * each.abs().sum(dim=1))
    assert not combine_rows(y, order)[5].any()
    gather_rows(normal(1, 20, 24), order)
    _, dw = combine_rows_backward(normal(1, 20, 24), y, order)
    assert float(dw[3, 0]) == float(dw[4, 1]) == 0 and not dw[5].any()
    for end in (-5, 2 ** 31 - 1):
        order.offs[-1] = end
        assert gather_rows(normal(1, 20, 24), order).shape == (40, 24)


def test_gradients_through_autograd():
    """The three differentiable calls in a chain, against the same formulas in 64 bits; expanded and transposed gradients."""
    from kernels import combine_rows, gather_rows, route_topk, sort_by_expert

    tokens, experts, k, h = 30, 16, 4, 40
    leaves = [normal(1, tokens, h), normal(2, tokens, experts)]
    x, logits = (leaf.clone().requires_grad_() for leaf in leaves)
    x64, logits64 = (leaf.double().requires_grad_() for leaf in leaves)
    weights, chosen = route_topk(logits, k, normalize=False)
    order = sort_by_expert(chosen, experts)
    scale = 1 + torch.arange(tokens * k, device="cuda")[:, None] / 100
    out = combine_rows(torch.tanh(gather_rows(x, order)) * scale, order, weights)
    w64 = torch.softmax(logits64, dim=1).gather(1, chosen.long())
    slots = order.slots.long()
    ys64 = torch.tanh(x64[slots // k]) * scale.double()
    out64 = (ys64[order.places.long()] * w64[..., None]).sum(dim=1)
    within(out, out64.detach(), 2.0 ** -16)
    for reduce in (lambda o: o.sum(), lambda o: (o.t() * torch.ones(h, 1, device="cuda", dtype=o.dtype)).sum(), lambda o: o[:, 3].sum()):
        for a, b in ((x, x64), (logits, logits64)):
            a.grad = b.grad = None
        reduce(out).backward(retain_graph=True)
        reduce(out64).backward(retain_graph=True)
        for a, b in ((x, x64), (logits, logits64)):
            within(a.grad, b.grad, 2.0 ** -16 * b.grad.abs().max())


def test_only_what_a_gradient_needs_is_kept():
    from kernels import combine_rows

    order = order_of(5, 12, 2, 4)
    y, w = normal(1, 24, 16).requires_grad_(), normal(2, 12, 2)
    out = combine_rows(y, order, w)
    with torch.no_grad():
        y.mul_(2.0)  # not read for its own gradient
    out.sum().backward()
    assert torch.equal(y.grad, w.flatten()[order.slots.long()][:, None].expand(24, 16))


def test_calls_on_another_stream_and_in_a_replayed_graph():
    from kernels import combine_rows, combine_rows_backward, gather_rows, route_topk, route_topk_backward, sort_by_expert

    x, logits = normal(1, 500, 264).to(torch.bfloat16), normal(2, 500, 64)
    dw = normal(3, 500, 4)

    def step():
        weights, chosen = route_topk(logits, 4)
        order = sort_by_expert(chosen, 64)
        xs = gather_rows(x, order)
        return (weights, *order, xs, combine_rows(xs, order, weights), *combine_rows_backward(x, xs, order, weights),
                route_topk_backward(dw, logits, chosen))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        there = step()
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in zip(there, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (7, 8, 9):
        x.copy_(normal(seed, 500, 264))
        logits.copy_(normal(seed + 10, 500, 64))
        expected = step()
        torch.cuda.synchronize()
        graph.replay()
        for a, b in zip(captured, expected):
            assert torch.equal(a, b)
