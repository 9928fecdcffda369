"""GPU tests of the Gate+Up training form (h, dx, dW) against its formulas in 64 bits.

Bounds (derived, elementwise), with u the half unit of the operand type and eps = 2^-23: the fp32 projections are
off by at most (H + 8) eps sum |x w|; silu' is at most 1.1 in size and silu'' at most 0.5; dP is computed in fp32
(2^-19 of its factors' sizes for exp, reciprocal and products) and rounded to the operand type (u |dP|, or the least
normal's unit); the two products add their own fp32 sums and one rounding.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALL = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
EPS = 2.0 ** -23


@pytest.fixture(autouse=True)
def _gpu_only():
    if not torch.cuda.is_available():
        pytest.skip("ROCm GPU unavailable")


def normal(seed, *shape):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def operands(seed, counts, h, f, dtype):
    rows = sum(counts)
    x = normal(seed, rows, h).to(dtype)
    w = (normal(seed + 1, len(counts), h, 2 * f) / h ** 0.5).to(dtype)
    dh = normal(seed + 2, rows, f).to(dtype)
    offs = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    return x, w, dh, offs


def within(actual, exact, bound):
    worst = float(((actual.double() - exact).abs() - bound).max()) if actual.numel() else -1.0
    assert torch.isfinite(actual).all() and worst <= 0, worst


def check_group(x, w, dh, h, saved, dx, dw):
    """One group's outputs against the formulas."""
    dtype, f = x.dtype, w.shape[1] // 2
    unit, small = HALF_UNIT[dtype], SMALL[dtype]
    x, w, dh = x.double(), w.double(), dh.double()
    p = x @ w
    p_error = (x.shape[1] + 8) * EPS * (x.abs() @ w.abs())
    if saved is not None:
        within(saved, p, p_error + 2.0 ** -40)
    g, u, ge, ue = p[:, :f], p[:, f:], p_error[:, :f], p_error[:, f:]
    s = torch.sigmoid(g)
    if h is not None:
        exact = g * s * u
        within(h, exact, unit * exact.abs() + 1.1 * u.abs() * ge + (g * s).abs() * ue + 1.1 * ge * ue
               + 2.0 ** -19 * exact.abs() + small)
    slope = s * (1 + g * (1 - s))
    dp = torch.cat([dh * u * slope, dh * g * s], dim=1)
    fp32 = torch.cat([dh.abs() * (0.5 * u.abs() * ge + slope.abs() * ue + 0.5 * ge * ue + 2.0 ** -19 * u.abs() * (1 + g.abs())),
                      dh.abs() * (1.1 * ge + 2.0 ** -19 * g.abs())], dim=1)
    dp_error = fp32 + unit * (dp.abs() + fp32) + small
    rounding = 2.0 ** -40 + small
    if dx is not None:
        exact = dp @ w.t()
        bound = dp_error @ w.abs().t() + (2 * f + 8) * EPS * ((dp.abs() + dp_error) @ w.abs().t())
        within(dx, exact, bound + unit * (exact.abs() + bound) + rounding)
    if dw is not None:
        exact = x.t() @ dp
        bound = x.abs().t() @ dp_error + (x.shape[0] + 8) * EPS * (x.abs().t() @ (dp.abs() + dp_error))
        within(dw, exact, bound + unit * (exact.abs() + bound) + rounding)


def check(x, w, dh, counts, h, saved, dx, dw):
    first = 0
    for e, count in enumerate(counts):
        part = slice(first, first + count)
        first += count
        if count:
            check_group(x[part], w[e], dh[part], None if h is None else h[part], None if saved is None else saved[part],
                        None if dx is None else dx[part], None if dw is None else dw[e])
        elif dw is not None:
            assert not dw[e].any()


SHAPES = [((1,), 8, 8), ((3, 0, 1), 64, 72), ((17, 40, 0, 5, 64), 264, 136), ((0, 0, 0), 128, 64), ((300, 1, 129), 520, 320),
          ((64,) * 8, 512, 512), ((2,) * 70, 40, 24), ((700, 0, 33), 1032, 264)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts,h,f", SHAPES)
def test_forward_and_backward_match_64_bits(counts, h, f, dtype):
    from kernels import gate_up_swiglu_backward, gate_up_swiglu_forward

    print(f"gate_up_swiglu counts={counts[:8]} h={h} f={f} {dtype}", flush=True)
    x, w, dh, offs = operands(sum(counts) + h, counts, h, f, dtype)
    out, saved = gate_up_swiglu_forward(x, w, offs)
    dx, dw = gate_up_swiglu_backward(dh, x, w, offs, saved)
    assert out.dtype == dx.dtype == dw.dtype == dtype and dw.shape == w.shape
    check(x, w, dh, counts, out, saved, dx, dw)


@pytest.mark.parametrize("counts,h,f", [((70, 0, 9, 200), 328, 200), ((31,), 264, 520)])
def test_every_variant_matches_64_bits(counts, h, f):
    from kernels import _native, gate_up_swiglu_backward, gate_up_swiglu_forward

    lib = _native.library()
    x, w, dh, offs = operands(9, counts, h, f, torch.bfloat16)
    out, saved = gate_up_swiglu_forward(x, w, offs)
    for product in range(3):
        for variant in range(lib.moegemm_gate_up_variant_count(product)):
            print(f"gate_up product={product} variant={variant} counts={counts}", flush=True)
            for _ in range(2):
                if product == 0:
                    got, kept = gate_up_swiglu_forward(x, w, offs, variant=variant)
                    check(x, w, dh, counts, got, kept, None, None)
                else:
                    dx, dw = gate_up_swiglu_backward(dh, x, w, offs, saved, need_dx=product == 1, need_dw=product == 2,
                                                     variants=(variant, variant))
                    check(x, w, dh, counts, None, None, dx, dw)


def test_rows_past_the_groups_are_zero_and_offsets_are_clamped():
    from kernels import gate_up_swiglu_backward, gate_up_swiglu_forward

    x, w, dh, _ = operands(3, (90, 0, 40), 136, 72, torch.bfloat16)
    for ends, counts in (([20, 20, 60], (20, 0, 40)), ([-3, 30, 1000], (0, 30, 100)), ([0, 0, 0], (0, 0, 0))):
        offs = torch.tensor(ends, dtype=torch.int32, device="cuda")
        end = sum(counts)
        torch.full((130, 400), float("nan"), device="cuda")  # a reused block would show unwritten rows
        out, saved = gate_up_swiglu_forward(x, w, offs)
        dx, dw = gate_up_swiglu_backward(dh, x, w, offs, saved)
        assert not out[end:].any() and not dx[end:].any()
        check(x, w, dh, counts, out, saved, dx, dw)


def test_one_group_strides_and_alignment():
    from kernels import gate_up_swiglu_backward, gate_up_swiglu_forward

    x, w, dh, _ = operands(5, (75,), 136, 72, torch.float16)
    out, saved = gate_up_swiglu_forward(x, w[0])
    dx, dw = gate_up_swiglu_backward(dh, x, w[0], None, saved)
    assert dw.shape == (136, 144)
    check(x, w, dh, (75,), out, saved, dx, dw[None])
    wide_x = torch.zeros((150, 160), device="cuda", dtype=torch.float16)[::2, 8:144]
    wide_w = torch.zeros((1, 136, 160), device="cuda", dtype=torch.float16)[:, :, 16:]
    wide_dh = torch.zeros((75, 80), device="cuda", dtype=torch.float16)[:, 8:]
    wide_x.copy_(x), wide_w.copy_(w), wide_dh.copy_(dh)
    offs = torch.tensor([75], dtype=torch.int32, device="cuda")
    out2, saved2 = gate_up_swiglu_forward(wide_x, wide_w, offs)
    assert torch.equal(out, out2) and torch.equal(saved, saved2)
    for grad in (wide_dh, dh.t().contiguous().t()):
        dx2, dw2 = gate_up_swiglu_backward(grad, wide_x, wide_w, offs, saved2)
        assert torch.equal(dx, dx2) and torch.equal(dw, dw2[0])
    for dx_only in (True, False):
        pair = gate_up_swiglu_backward(dh, x, w[0], None, saved, need_dx=dx_only, need_dw=not dx_only)
        assert (pair[0] is None) != dx_only and (pair[1] is None) == dx_only


def test_autograd_gives_the_same_gradients_and_matches_differences():
    from kernels import gate_up_swiglu, gate_up_swiglu_backward, gate_up_swiglu_forward

    counts = (40, 0, 25)
    x, w, dh, offs = operands(7, counts, 64, 40, torch.bfloat16)
    x1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
    h = gate_up_swiglu(x1, w1, offs)
    h.backward(dh)
    _, saved = gate_up_swiglu_forward(x, w, offs)
    dx, dw = gate_up_swiglu_backward(dh, x, w, offs, saved)
    assert torch.equal(x1.grad, dx) and torch.equal(w1.grad, dw)
    gate_up_swiglu(x1, w1, offs).sum().backward()  # an expanded gradient

    def loss(x64, w64):
        total, first = 0.0, 0
        for e, count in enumerate(counts):
            p = x64[first:first + count] @ w64[e]
            first += count
            total = total + ((p[:, :40] * torch.sigmoid(p[:, :40]) * p[:, 40:]) * dh[first - count:first].double()).sum()
        return total

    # Central differences of the 64-bit loss along random directions: the second-order term is 1e-10 of the
    # loss, so what is left is the gradients' own rounding, u per element and independent.
    for seed in range(3):
        vx, vw = normal(seed, *x.shape).double(), normal(seed + 50, *w.shape).double()
        step = 1e-5
        slope = (loss(x.double() + step * vx, w.double() + step * vw)
                 - loss(x.double() - step * vx, w.double() - step * vw)) / (2 * step)
        along = (dx.double() * vx).sum() + (dw.double() * vw).sum()
        spread = float(((dx.double() * vx).norm() ** 2 + (dw.double() * vw).norm() ** 2) ** 0.5)
        assert abs(float(along - slope)) <= 8 * 2.0 ** -8 * spread


def test_extreme_gates_keep_finite_gradients():
    from kernels import gate_up_swiglu_backward, gate_up_swiglu_forward

    x = torch.ones((4, 8), device="cuda", dtype=torch.bfloat16)
    w = torch.zeros((8, 16), device="cuda", dtype=torch.bfloat16)
    w[0, :8] = torch.tensor([200.0, -200.0, 1e4, -1e4, 88.0, -88.0, 0.0, 1e-30])
    w[0, 8:] = 1.0
    out, saved = gate_up_swiglu_forward(x, w)
    dx, dw = gate_up_swiglu_backward(torch.ones_like(out), x, w, None, saved)
    assert all(torch.isfinite(t).all() for t in (out, dx, dw))
    check_group(x, w, torch.ones_like(out), out, saved, dx, dw)
    x[2, 3] = float("nan")
    out, saved = gate_up_swiglu_forward(x, w)
    assert torch.isnan(out[2]).all() and torch.isfinite(out[[0, 1, 3]]).all()


def test_graph_replays_read_new_offsets():
    from kernels import gate_up_swiglu_backward, gate_up_swiglu_forward

    x, w, dh, offs = operands(11, (30, 34, 0, 36), 136, 72, torch.bfloat16)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        gate_up_swiglu_backward(dh, x, w, offs, gate_up_swiglu_forward(x, w, offs)[1])
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out, saved = gate_up_swiglu_forward(x, w, offs)
        dx, dw = gate_up_swiglu_backward(dh, x, w, offs, saved)
    for ends in ([30, 64, 64, 100], [100, 100, 100, 100], [0, 1, 50, 80]):
        offs.copy_(torch.tensor(ends, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        eager, kept = gate_up_swiglu_forward(x, w, offs)
        edx, edw = gate_up_swiglu_backward(dh, x, w, offs, kept)
        assert torch.equal(out, eager) and torch.equal(dx, edx) and torch.equal(dw, edw)


def test_rows_past_two_gib_of_one_expert():
    """One expert's rows span more than 2 GiB: dW's K runs in segments."""
    from kernels import gate_up_swiglu_backward, gate_up_swiglu_forward

    rows, h, f = 140_000, 8192, 16
    x = torch.zeros((rows, h), device="cuda", dtype=torch.bfloat16)  # 2.3 GB
    keep = [0, 65_535, 65_536, 131_072, rows - 1]
    x[keep] = normal(13, 5, h).to(torch.bfloat16)
    w = (normal(14, 2, h, 2 * f) / h ** 0.5).to(torch.bfloat16)
    dh = normal(15, rows, f).to(torch.bfloat16)
    offs = torch.tensor([rows, rows], dtype=torch.int32, device="cuda")
    out, saved = gate_up_swiglu_forward(x, w, offs)
    dx, dw = gate_up_swiglu_backward(dh, x, w, offs, saved)
    # Rows of zeros have g = u = 0, so h, dP and their share of dW are exactly zero.
    check_group(x[keep], w[0], dh[keep], out[keep], saved[keep], dx[keep], dw[0])
    assert not dw[1].any() and not out[1:65_535].any() and not dx[1:65_535].any()


def test_more_groups_than_a_launch_lists():
    """Over 768 experts: several launches; the groups around each launch's ends are checked."""
    from kernels import _native, gate_up_swiglu_backward, gate_up_swiglu_forward

    lib = _native.library()
    counts = [(i * 7) % 3 for i in range(1100)]
    x, w, dh, offs = operands(5, counts, 24, 16, torch.bfloat16)
    starts = offs.tolist()
    for variant in (None, *range(lib.moegemm_gate_up_variant_count(0))):
        print(f"gate_up 1100 experts variant={variant}", flush=True)
        out, saved = gate_up_swiglu_forward(x, w, offs, variant=variant)
        back = min(variant or 0, lib.moegemm_gate_up_variant_count(2) - 1)
        dx, dw = gate_up_swiglu_backward(dh, x, w, offs, saved, variants=None if variant is None else (variant, back))
        for e in [*range(0, 12), *range(760, 776), *range(1090, 1100)]:
            part = slice(starts[e] - counts[e], starts[e])
            if counts[e]:
                check_group(x[part], w[e], dh[part], out[part], saved[part], dx[part], dw[e])
            else:
                assert not dw[e].any()


def test_more_rounds_than_a_launch_lists(monkeypatch):
    """More than 192 tiles on one workgroup: the launches after the first start where it ended."""
    from kernels import _native, gated_ffn

    lib = _native.library()
    counts = (20, 0, 50)
    x, w, dh, offs = operands(6, counts, 264, 128 * 140, torch.bfloat16)
    out, saved = gated_ffn.gate_up_swiglu_forward(x, w, offs)
    dx, dw = gated_ffn.gate_up_swiglu_backward(dh, x, w, offs, saved)
    monkeypatch.setattr(gated_ffn, "_cu_count", lambda *_: 1)
    close = dict(rtol=2.0 ** -6, atol=2.0 ** -6)
    for variant in range(lib.moegemm_gate_up_variant_count(0)):
        print(f"gate_up forward one workgroup variant={variant}", flush=True)
        got, kept = gated_ffn.gate_up_swiglu_forward(x, w, offs, variant=variant)
        torch.testing.assert_close(got, out, **close)
        torch.testing.assert_close(kept, saved, rtol=1e-5, atol=1e-4)
    for variant in range(lib.moegemm_gate_up_variant_count(2)):
        print(f"gate_up dw one workgroup variant={variant}", flush=True)
        _, got = gated_ffn.gate_up_swiglu_backward(dh, x, w, offs, saved, need_dx=False, variants=(variant, variant))
        torch.testing.assert_close(got, dw, **close)


def test_a_gradient_broadcast_over_rows():
    """The gradient of h.sum(0) reaches the block with strides (0, 1): every row is the same one."""
    from kernels import gate_up_swiglu, gate_up_swiglu_backward, gate_up_swiglu_forward

    x, w, dh, offs = operands(17, (40, 0, 25), 64, 40, torch.bfloat16)
    x1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
    v = dh[0].clone()
    gate_up_swiglu(x1, w1, offs).sum(0).backward(v)
    _, saved = gate_up_swiglu_forward(x, w, offs)
    dx, dw = gate_up_swiglu_backward(v.repeat(65, 1), x, w, offs, saved)
    assert torch.equal(x1.grad, dx) and torch.equal(w1.grad, dw)
    overlapping = torch.as_strided(normal(18, 65 * 8 + 40).to(torch.bfloat16), (65, 40), (8, 1))
    pair = gate_up_swiglu_backward(overlapping, x, w, offs, saved)
    dense = gate_up_swiglu_backward(overlapping.clone(), x, w, offs, saved)
    assert torch.equal(pair[0], dense[0]) and torch.equal(pair[1], dense[1])


def test_a_gradient_at_an_odd_offset():
    """The gradient of a concatenation is a view of a larger buffer: dense, but not on a multiple of 16 bytes."""
    from kernels import gate_up_swiglu, gate_up_swiglu_backward, gate_up_swiglu_forward

    x, w, dh, offs = operands(19, (40, 0, 25), 64, 40, torch.float16)
    x1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
    odd = torch.zeros(3, device="cuda", dtype=torch.float16)
    torch.cat([odd, gate_up_swiglu(x1, w1, offs).flatten()]).backward(torch.cat([odd, dh.flatten()]))
    _, saved = gate_up_swiglu_forward(x, w, offs)
    dx, dw = gate_up_swiglu_backward(dh, x, w, offs, saved)
    assert torch.equal(x1.grad, dx) and torch.equal(w1.grad, dw)


def test_only_what_a_gradient_needs_is_kept():
    """An operand that no wanted gradient reads may change, or be freed, before the backward pass."""
    from kernels import gate_up_swiglu, gate_up_swiglu_backward, gate_up_swiglu_forward

    x, w, dh, offs = operands(23, (40, 0, 25), 64, 40, torch.bfloat16)
    _, saved = gate_up_swiglu_forward(x, w, offs)
    dx, dw = gate_up_swiglu_backward(dh, x, w, offs, saved)
    x1, w1 = x.clone().requires_grad_(), w.clone()
    h = gate_up_swiglu(x1, w1, offs)
    with torch.no_grad():
        x1.zero_()  # dx is dP W^T
    h.backward(dh)
    assert torch.equal(x1.grad, dx) and w1.grad is None
    x1, w1 = x.clone(), w.clone().requires_grad_()
    h = gate_up_swiglu(x1, w1, offs)
    with torch.no_grad():
        w1.zero_()  # dW is x^T dP
    h.backward(dh)
    assert torch.equal(w1.grad, dw) and x1.grad is None


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_no_projections_are_kept_without_a_gradient(dtype):
    """Without a gradient to come h is the same bits, and its rows are all that is allocated."""
    from kernels import _native, gate_up_swiglu, gate_up_swiglu_forward

    for counts, h, f in (((2,), 64, 72), ((300, 0, 129), 520, 320), ((1000, 600), 256, 1024)):
        x, w, _, offs = operands(29, counts, h, f, dtype)
        expected, _ = gate_up_swiglu_forward(x, w, offs)
        w.requires_grad_()
        for enabled, weight in ((False, w), (True, w.detach())):
            torch.cuda.synchronize()
            before = torch.cuda.memory_allocated()
            torch.cuda.reset_peak_memory_stats()
            with torch.set_grad_enabled(enabled):
                out = gate_up_swiglu(x, weight, offs)
            assert torch.cuda.max_memory_allocated() - before <= -(-out.numel() * 2 // 512) * 512
            assert torch.equal(out, expected) and not out.requires_grad
    lib = _native.library()
    for variant in range(lib.moegemm_gate_up_variant_count(0)):  # the C entry keeps nothing where saved is null
        out = torch.full_like(expected, float("nan"))
        _native.check(lib.moegemm_gate_up_forward(
            x.data_ptr(), w.data_ptr(), out.data_ptr(), None, offs.data_ptr(), 2, 1600, 256, 1024, 256, 256 * 2048, 2048,
            1024, _native.dtype_code(dtype), variant, 256, _native.current_stream_handle(x.device)))
        assert torch.equal(out, gate_up_swiglu_forward(x, w, offs, variant=variant)[0])


def poison(*shapes_and_types):
    """Blocks of NaN that the next allocations of the same sizes reuse: rows that stay unwritten show."""
    blocks = [torch.full(shape, float("nan"), device="cuda", dtype=dtype) for shape, dtype in shapes_and_types]
    del blocks


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cus", [1, 3, 8])
def test_widest_tiles_chained_over_few_workgroups(cus, dtype, monkeypatch):
    """Several 256x256 tiles a workgroup in all three products: dW's K is 5, 10, 4 and 2 slices of 32 rows, so that tiles
    with a prefetched successor and ones too short for it alternate."""
    from kernels import gated_ffn

    counts, h, f = (130, 0, 300, 97, 64), 520, 320
    x, w, dh, offs = operands(31, counts, h, f, dtype)
    rows = sum(counts)
    monkeypatch.setattr(gated_ffn, "_cu_count", lambda *_: cus)
    for ends in (counts, (0, 64, 33, 0, 300)):
        offs = torch.tensor(ends, device="cuda").cumsum(0).to(torch.int32)
        end = sum(ends)
        print(f"chained tiles cus={cus} counts={ends} {dtype}", flush=True)
        poison(((rows, f), dtype), ((rows, 2 * f), torch.float32))
        out, saved = gated_ffn.gate_up_swiglu_forward(x, w, offs, variant=0)
        check(x, w, dh, ends, out, saved, None, None)
        poison(((rows, 2 * f), dtype), ((rows, h), dtype), (w.shape, dtype))
        dx, dw = gated_ffn.gate_up_swiglu_backward(dh, x, w, offs, saved, variants=(0, 0))
        check(x, w, dh, ends, None, None, dx, dw)
        assert not out[end:].any() and not dx[end:].any()


@pytest.mark.parametrize("cus,h,f", [(8, 256, 128), (5, 256, 128), (8, 64, 72), (8, 520, 200), (16, 256, 128)])
def test_short_last_rounds_are_shared_by_rows(cus, h, f, monkeypatch):
    """One full round of 256x256 tiles and 1 to 4 tiles more, whose rows go to two or four workgroups: tiles of every
    kind of row count, one and several columns of tiles, behind chained tiles (H 256 and 520) and unchained ones (H 64)."""
    from kernels import gated_ffn

    monkeypatch.setattr(gated_ffn, "_cu_count", lambda *_: cus)
    for last in ((1,), (63,), (64,), (65,), (129,), (256,), (129, 65), (1, 256), (63, 64, 129), (256, 1, 65), (193, 0, 128, 2, 250)):
        counts = (256,) * cus + last
        rows = sum(counts)
        x, w, dh, offs = operands(37 + sum(last), counts, h, f, torch.bfloat16)
        print(f"short last round cus={cus} h={h} f={f} last={last}", flush=True)
        poison(((rows, f), x.dtype), ((rows, 2 * f), torch.float32))
        out, saved = gated_ffn.gate_up_swiglu_forward(x, w, offs, variant=0)
        poison(((rows, 2 * f), x.dtype), ((rows, h), x.dtype))
        dx, _ = gated_ffn.gate_up_swiglu_backward(dh, x, w, offs, saved, need_dw=False, variants=(0, 0))
        check(x, w, dh, counts, out, saved, dx, None)


def test_weights_past_32_bit_offsets():
    """Experts whose weights and gradients start past 4 GiB."""
    from kernels import gate_up_swiglu_backward, gate_up_swiglu_forward

    groups, h, f = 5, 4096, 65536  # 1.07 GB an expert
    x = normal(41, 7, h).to(torch.bfloat16)
    w = torch.empty((groups, h, 2 * f), device="cuda", dtype=torch.bfloat16)
    for e in range(groups):
        w[e] = normal(42 + e, h, 2 * f) / h ** 0.5
    dh = normal(47, 7, f).to(torch.bfloat16)
    offs = torch.tensor([2, 2, 2, 2, 7], dtype=torch.int32, device="cuda")
    out, saved = gate_up_swiglu_forward(x, w, offs)
    dx, dw = gate_up_swiglu_backward(dh, x, w, offs, saved)
    check_group(x[2:], w[4], dh[2:], out[2:], saved[2:], dx[2:], dw[4])
    assert not dw[1:4].any()


def test_rows_past_32_bit_offsets():
    """Rows 8 MB apart: x and dh pass 4 GiB, and dW's K runs in segments of 128 rows."""
    from kernels import _native, gate_up_swiglu_backward, gate_up_swiglu_forward

    lib = _native.library()
    pitch, counts, h, f = (1 << 22) - 8, (300, 0, 400), 72, 40
    x, w, dh, offs = operands(53, counts, h, f, torch.bfloat16)
    wide = torch.zeros((700, pitch), device="cuda", dtype=torch.bfloat16)  # 5.9 GB
    far_x, far_dh = wide[:, :h], wide[:, 80:80 + f]
    far_x.copy_(x), far_dh.copy_(dh)
    for variant in range(lib.moegemm_gate_up_variant_count(0)):
        print(f"rows 8 MB apart variant={variant}", flush=True)
        out, saved = gate_up_swiglu_forward(far_x, w, offs, variant=variant)
        back = min(variant, lib.moegemm_gate_up_variant_count(2) - 1)
        dx, dw = gate_up_swiglu_backward(far_dh, far_x, w, offs, saved, variants=(variant, back))
        check(x, w, dh, counts, out, saved, dx, dw)


def test_a_gradient_sliced_from_a_wide_one():
    """h beside four million other columns: its gradient's rows are 8 MB apart."""
    from kernels import gate_up_swiglu, gate_up_swiglu_backward, gate_up_swiglu_forward

    x, w, dh, offs = operands(59, (3, 0, 2), 64, 40, torch.bfloat16)
    x1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
    other = torch.zeros((5, 1 << 22), device="cuda", dtype=torch.bfloat16)
    torch.cat([gate_up_swiglu(x1, w1, offs), other], dim=1).backward(torch.cat([dh, other], dim=1))
    _, saved = gate_up_swiglu_forward(x, w, offs)
    dx, dw = gate_up_swiglu_backward(dh, x, w, offs, saved)
    assert torch.equal(x1.grad, dx) and torch.equal(w1.grad, dw)
