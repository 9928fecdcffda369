"""GPU tests of the 4-bit (MXFP4) operators against their definitions in 64 bits.

Bounds (derived, elementwise).  Conversions are exact: quantised bytes equal the definition's, and values equal them in
bf16 and fp32 (fp16: one rounding).  Products: a weight is exact in bf16 and a row is a sum of exact bf16 parts, so an output
differs from the 64-bit sum by the fp32 sums' rounding alone, (K + 8) 2^-23 sum_k |a w| (a unit of 2^-23 covers
truncating adds), plus half a unit of the output type.  fp32 rows are two bf16 parts: the first is cut to 8 bits, which leaves less than
2^-7 of a value, of which the second keeps all but 2^-9: 2^-16 sum_k |a w| more.  Gate+Up: silu' is at most 1.1 in size, and exp, division and
products in fp32 round by 2^-19 of the result.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SMALL = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


@pytest.fixture(autouse=True)
def _gpu_only():
    if not torch.cuda.is_available():
        pytest.skip("ROCm GPU unavailable")


def normal(seed, *shape):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def values(q, scale):
    """64-bit values of packed bytes."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device=q.device)
    code = torch.stack([q & 15, q >> 4], dim=-1).reshape(*scale.shape, 32)
    factor = torch.where(scale == 255, float("nan"), torch.exp2(scale.double() - 127))
    return (table[code.long()] * factor[..., None]).reshape(*scale.shape[:-1], -1)


def weight(seed, *shape, low=115, high=125):
    """Random codes and scales of a weight [..., K]."""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    *head, k = shape
    q = torch.randint(0, 256, (*head, k // 2), device="cuda", dtype=torch.uint8, generator=generator)
    return q, torch.randint(low, high, (*head, k // 32), device="cuda", dtype=torch.uint8, generator=generator)


def sums(a):
    """Error of a sum of products per sum of their sizes."""
    return (a.shape[1] + 8) * 2.0 ** -23 + (2.0 ** -16 if a.dtype is torch.float32 else 0.0)


def close(out, a, w, extra=0.0):
    """``out`` against a @ w.T, elementwise."""
    x = a.double()
    exact, size = x @ w.t(), x.abs() @ w.abs().t()
    bound = HALF_UNIT[out.dtype] * exact.abs() + sums(a) * size + SMALL[out.dtype] + extra
    worst = float(((out.double() - exact).abs() - bound).max()) if out.numel() else -1.0
    assert torch.isfinite(out).all() and worst <= 0, worst


def close_gated(h, a, w):
    x, f = a.double(), w.shape[0] // 2
    p, size = x @ w.t(), sums(a) * (x.abs() @ w.abs().t())
    g, u, ge, ue = p[:, :f], p[:, f:], size[:, :f], size[:, f:]
    s = torch.sigmoid(g)
    exact = g * s * u
    bound = (HALF_UNIT[h.dtype] + 2.0 ** -19) * exact.abs() + 1.1 * u.abs() * ge + (g * s).abs() * ue + 1.1 * ge * ue
    worst = float(((h.double() - exact).abs() - bound - SMALL[h.dtype]).max()) if h.numel() else -1.0
    assert torch.isfinite(h).all() and worst <= 0, worst


def quantised(x):
    """(codes packed, scales) by the definition, on the CPU in 64 bits."""
    blocks = x.double().cpu().reshape(*x.shape[:-1], -1, 32)
    top = blocks.abs().amax(dim=-1)
    exponent = torch.where(top > 0, torch.frexp(top).exponent.long() - 3, -127).clamp(min=-127)
    size = (blocks.abs() * torch.exp2(-exponent.double())[..., None]).clamp(max=6)
    grid = torch.tensor(E2M1, dtype=torch.float64)
    code = (size[..., None] - grid).abs()
    code = torch.where(code == code.amin(dim=-1, keepdim=True), torch.arange(8), 99)
    low, high = code.amin(dim=-1), torch.where(code == 99, -1, code).amax(dim=-1)
    code = torch.where(low % 2 == 0, low, high)  # a tie goes to the even code
    code = (code + 8 * torch.signbit(blocks)).reshape(*x.shape[:-1], -1, 2).to(torch.uint8)
    return code[..., 0] | code[..., 1] << 4, (exponent + 127).to(torch.uint8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 32), (3, 64), (17, 2880), (130, 992), (2, 5, 96), (8, 100, 512)])
def test_quantize_matches_the_definition(shape, dtype):
    from kernels import dequantize_mxfp4, quantize_mxfp4

    x = (normal(shape[-1], *shape) * normal(7, *shape[:-1], 1).exp()).to(dtype)
    x[..., :32] = 0
    x[..., 0, 0] = -0.0
    x[..., -16:] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -0.75, -1.25, -2.5, -5.0, 4.0, 6.5, -7.9]).to(dtype)
    q, scale = quantize_mxfp4(x)
    codes, scales = quantised(x)
    assert torch.equal(scale.cpu(), scales) and torch.equal(q.cpu(), codes)
    for out in (torch.bfloat16, torch.float16, torch.float32):
        back = dequantize_mxfp4(q, scale, dtype=out)
        assert back.dtype is out and torch.equal(back, values(q, scale).to(out))
    assert dequantize_mxfp4(q, scale).dtype is torch.bfloat16


def test_quantize_extremes():
    from kernels import dequantize_mxfp4, quantize_mxfp4

    x = normal(3, 8, 64)
    for factor in (2.0 ** 120, 2.0 ** -120, 2.0 ** -126):
        q, scale = quantize_mxfp4(x * factor)
        codes, scales = quantised(x * factor)
        assert torch.equal(scale.cpu(), scales) and torch.equal(q.cpu(), codes)
    for bad in (float("nan"), float("inf"), -float("inf")):
        y = x.clone()
        y[2, 40] = bad
        q, scale = quantize_mxfp4(y)
        back = dequantize_mxfp4(q, scale)
        assert int(scale[2, 1]) == 255 and torch.isnan(back[2, 32:]).all() and int(torch.isnan(back).sum()) == 32


def test_every_code_and_scale_comes_back():
    from kernels import dequantize_mxfp4

    q = torch.arange(256, device="cuda", dtype=torch.uint8).repeat(256, 1)  # [256, 512]: every pair under every scale
    scale = torch.arange(256, device="cuda", dtype=torch.uint8)[:, None].repeat(1, 16)
    exact = values(q, scale)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        torch.testing.assert_close(dequantize_mxfp4(q, scale, dtype=dtype), exact.to(dtype), rtol=0, atol=0, equal_nan=True)


def test_conversion_strides():
    from kernels import dequantize_mxfp4, quantize_mxfp4

    base = normal(3, 6, 50, 900).to(torch.bfloat16)
    for view in (base[:, 3:, 1:641], base[:, 7:8, :32], base[:1, :3, :64].expand(5, 3, 64), base[::2, ::3, :96], base[4, :, :64], base[:1, :, 8:40], base[:, :0, :32]):
        q, scale = quantize_mxfp4(view)
        q0, scale0 = quantize_mxfp4(view.contiguous())
        assert torch.equal(q, q0) and torch.equal(scale, scale0)
    q, scale = weight(2, 7, 20, 320)
    for part in ((slice(1, 5), slice(2, 18)), (slice(None), slice(0, 1)), (slice(2, 3), slice(None))):
        a, b = q[part][..., 32:96], scale[part][..., 2:6]
        assert torch.equal(dequantize_mxfp4(a, b), dequantize_mxfp4(a.contiguous(), b.contiguous()))
    x = normal(1, 4, 32).t().contiguous().t()
    with pytest.raises(ValueError, match="unit stride"):
        quantize_mxfp4(x)


def _variants():
    from kernels import _native

    return [None, *range(_native.library().moegemm_mxfp4_variant_count())]


SHAPES = [(1, 1, 32), (1, 5760, 2880), (2, 40, 64), (5, 72, 160), (8, 130, 2880), (9, 257, 1056), (16, 64, 512), (17, 100, 7168),
          (33, 33, 288), (70, 96, 256)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_single_products(m, n, k, dtype):
    from kernels import grouped_mm_mxfp4_swiglu, matmul_mxfp4

    a = (normal(m + n, m, k) * normal(5, k).exp()).to(dtype)
    q, scale = weight(k, n, k)
    gate, gate_scale = weight(k + 1, 2 * n, k, high=118)
    w, wide = values(q, scale), values(gate, gate_scale)
    for variant in _variants():
        close(matmul_mxfp4(a, q, scale, variant=variant), a, w)
        close_gated(grouped_mm_mxfp4_swiglu(a, gate, gate_scale, variant=variant, out_dtype=torch.float32), a, wide)
    for out_dtype in (torch.float32, torch.float16, torch.bfloat16):
        if out_dtype is not torch.float16 or k < 1000:
            out = matmul_mxfp4(a, q, scale, out_dtype=out_dtype)
            assert out.dtype is out_dtype
            close(out, a, w)


GROUPS = [[1], [0, 3, 0, 5], [4, 0, 0, 1, 17, 2], [8] * 32, [0] * 9 + [1] + [0] * 5, [70, 1, 33, 0], [1] * 200, [0, 0]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("counts", GROUPS)
@pytest.mark.parametrize("n,k", [(48, 96), (130, 544)])
def test_grouped_products(counts, n, k, dtype):
    from kernels import grouped_mm_mxfp4, grouped_mm_mxfp4_swiglu

    rows = sum(counts)
    spare = 3
    a = normal(rows, rows + spare, k).to(dtype)
    a[rows:] = float("nan")  # rows behind the last group are not read
    q, scale = weight(n, len(counts), n, k)
    offs = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    w = values(q, scale)
    for variant in _variants():
        out = torch.full((rows + spare, n), 7.0, device="cuda", dtype=dtype)
        h = torch.full((rows + spare, n // 2), 7.0, device="cuda", dtype=torch.float32)
        assert grouped_mm_mxfp4(a, q, scale, offs, out=out, variant=variant) is out
        assert grouped_mm_mxfp4_swiglu(a, q, scale, offs, out=h, variant=variant) is h
        assert (out[rows:] == 7).all() and (h[rows:] == 7).all()
        first = 0
        for e, count in enumerate(counts):
            part = slice(first, first + count)
            close(out[part], a[part], w[e])
            close_gated(h[part], a[part], w[e])
            first += count


def test_more_groups_than_a_launch_takes():
    from kernels import grouped_mm_mxfp4

    counts = [(e * 7) % 3 for e in range(1700)]
    a = normal(1, sum(counts), 64).to(torch.bfloat16)
    q, scale = weight(4, 1700, 24, 64)
    offs = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    out = grouped_mm_mxfp4(a, q, scale, offs, out_dtype=torch.float32)
    owner = torch.arange(1700, device="cuda").repeat_interleave(torch.tensor(counts, device="cuda"))
    w, x = values(q, scale)[owner], a.double()
    exact, size = (w * x[:, None]).sum(dim=2), (w * x[:, None]).abs().sum(dim=2)
    assert bool(((out.double() - exact).abs() <= 72 * 2.0 ** -23 * size + 2.0 ** -23 * exact.abs()).all())


def test_offsets_past_the_rows_and_decreasing_ones_stay_in_bounds():
    from kernels import grouped_mm_mxfp4

    a = normal(1, 10, 96).to(torch.bfloat16)
    q, scale = weight(2, 4, 40, 96)
    w = values(q, scale)
    offs = torch.tensor([3, 8, 2 ** 31 - 1, 2 ** 31 - 1], device="cuda", dtype=torch.int32)
    out = grouped_mm_mxfp4(a, q, scale, offs)
    for e, (lo, hi) in enumerate(((0, 3), (3, 8), (8, 10), (10, 10))):
        close(out[lo:hi], a[lo:hi], w[e])
    for values_ in ([5, 2, 9, 1], [-4, -1, 3, 3]):
        grouped_mm_mxfp4(a, q, scale, torch.tensor(values_, device="cuda", dtype=torch.int32))
    torch.cuda.synchronize()
    # A group that begins before the end of an earlier, larger one: rows 2 to 90 are the third's or the first's.
    a = normal(3, 100, 96).to(torch.bfloat16)
    for variant in _variants():
        out = torch.zeros(100, 40, device="cuda", dtype=torch.bfloat16)
        grouped_mm_mxfp4(a, q, scale, torch.tensor([100, 2, 90, 1], device="cuda", dtype=torch.int32), out=out, variant=variant)
        close(out[:2], a[:2], w[0])
        close(out[90:], a[90:], w[0])
        assert torch.isfinite(out).all()


def test_scales_at_both_ends_and_nan():
    """Weights down to 2^-128 and up to 6 * 2^100, rows that bring the products back; a NaN scale reaches its column only."""
    from kernels import matmul_mxfp4

    for low, factor in ((0, 2.0 ** 100), (225, 2.0 ** -110)):
        q, scale = weight(low, 40, 256, low=low, high=low + 3)
        a = (normal(1, 6, 256) * factor).to(torch.bfloat16)
        close(matmul_mxfp4(a, q, scale, out_dtype=torch.float32), a, values(q, scale))
    q, scale = weight(9, 40, 320)
    scale[13, 4] = 255
    a = normal(2, 3, 320).to(torch.float16)
    out = matmul_mxfp4(a, q, scale)
    assert torch.isnan(out[:, 13]).all() and int(torch.isnan(out).sum()) == 3


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fp16_rows_keep_all_their_bits(dtype):
    """Single products of 1: every finite value of the row comes back in fp32, subnormals among them."""
    from kernels import matmul_mxfp4

    every = torch.arange(-2 ** 15, 2 ** 15, device="cuda", dtype=torch.int32).to(torch.int16).view(dtype)
    every = every[torch.isfinite(every)]
    count = len(every) // 32 * 32
    q = torch.zeros(32, 16, dtype=torch.uint8, device="cuda")
    for i in range(32):
        q[i, i // 2] = 2 << (4 * (i % 2))  # 1.0 on the diagonal
    out = matmul_mxfp4(every[:count].view(-1, 32), q, torch.full((32, 1), 127, dtype=torch.uint8, device="cuda"),
                       out_dtype=torch.float32)
    assert torch.equal(out.flatten(), every[:count].float())


def test_infinities_and_nan_stay_in_their_row():
    from kernels import matmul_mxfp4

    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        a = normal(4, 11, 288).abs().to(dtype)
        q, scale = weight(6, 50, 288)
        q &= 0x77  # no negative weights: an infinity cannot meet its opposite
        q |= 0x11  # nor a zero
        clean = matmul_mxfp4(a, q, scale)
        a[3, 100], a[7, 287] = float("inf"), float("nan")
        out = matmul_mxfp4(a, q, scale)
        assert (out[3] == float("inf")).all() and torch.isnan(out[7]).all()
        keep = [r for r in range(11) if r not in (3, 7)]
        assert torch.equal(out[keep], clean[keep])


def test_signalling_nans_and_infinities_in_every_variant():
    """The parts of a value that is no number give back what it is: in each kernel that splits rows, and in the one that does not."""
    from kernels import matmul_mxfp4

    q = torch.full((40, 48), 0x22, dtype=torch.uint8, device="cuda")  # 1.0 throughout
    scale = torch.full((40, 3), 127, dtype=torch.uint8, device="cuda")
    for dtype, whole, signalling in ((torch.float32, torch.int32, (0x7F800001, -0x7FFFFF)), (torch.float16, torch.int16, (0x7C01, -0x3FF)),
                                     (torch.bfloat16, torch.int16, (0x7F81, -0x7F))):
        for variant in _variants():
            a = torch.ones(6, 96, dtype=dtype, device="cuda")
            a[1, 7], a[2, 95] = float("inf"), -float("inf")
            a[3, 64], a[4, 31] = torch.tensor(signalling, dtype=whole, device="cuda").view(dtype)
            out = matmul_mxfp4(a, q, scale, variant=variant)
            assert (out[[0, 5]] == 96).all() and (out[1] == float("inf")).all() and (out[2] == -float("inf")).all()
            assert torch.isnan(out[3:5]).all()


def test_fp32_rows_from_end_to_end_of_their_range():
    """Values next to the largest and subnormal ones, and a NaN whose payload lies below bf16's bits."""
    from kernels import matmul_mxfp4

    a = torch.zeros(4, 64, device="cuda")
    a[0, 3], a[1, 40], a[2, 5] = torch.finfo(torch.float32).max, -2.0 ** -140, 1 + 2.0 ** -15
    a[3, 9] = torch.tensor(0x7f800001, dtype=torch.int32).view(torch.float32)
    q = torch.full((8, 32), 0x22, dtype=torch.uint8, device="cuda")  # 1.0 throughout
    out = matmul_mxfp4(a, q, torch.full((8, 2), 127, dtype=torch.uint8, device="cuda"))
    exact = a.double().sum(dim=1, keepdim=True)
    assert torch.isnan(out[3]).all()
    # The second part is a multiple of bf16's least number, 2^-133, and rounded to it: 2^-134 at most, here of one value times 1.
    # (Of a subnormal value the first part is 0 or such a multiple too, and nothing bounds the error by its size.)
    assert bool(((out[:3].double() - exact[:3]).abs() <= 2.0 ** -16 * exact[:3].abs() + 2.0 ** -134).all())
    wide = normal(2, 6, 130)[:, 2:98]  # rows at multiples of 8 bytes: refused
    with pytest.raises(ValueError, match="16 bytes"):
        matmul_mxfp4(wide, *weight(1, 8, 96))
    a = normal(2, 6, 132)[:, 4:100]
    close(matmul_mxfp4(a, *weight(1, 8, 96)), a, values(*weight(1, 8, 96)))


def test_one_rounding_with_a_wide_intermediate():
    """h in fp32 between the two products: off the 64-bit layer by one bf16 rounding, 2^-16 of each product's sizes and sums."""
    from kernels import grouped_mm_mxfp4, grouped_mm_mxfp4_swiglu

    a, offs = normal(1, 20, 160).to(torch.bfloat16), torch.tensor([12, 20], device="cuda", dtype=torch.int32)
    w13, w2 = weight(2, 2, 192, 160, low=118, high=121), weight(3, 2, 40, 96)
    h = grouped_mm_mxfp4_swiglu(a, *w13, offs, out_dtype=torch.float32)
    out = grouped_mm_mxfp4(h, *w2, offs, out_dtype=torch.bfloat16)
    for e, part in enumerate((slice(0, 12), slice(12, 20))):
        close_gated(h[part], a[part], values(*w13)[e])
        close(out[part], h[part], values(*w2)[e])
    assert out.dtype is torch.bfloat16


def test_strides_types_and_given_outputs():
    from kernels import grouped_mm_mxfp4, matmul_mxfp4

    a = normal(1, 12, 400).to(torch.bfloat16)[:, 8:328]
    q, scale = weight(3, 3, 60, 640)
    part, s = q[:, 5:50, 32:192], scale[:, 5:50, 2:12]
    offs = torch.tensor([4, 4, 12], device="cuda", dtype=torch.int32)
    wide = torch.zeros(12, 100, device="cuda", dtype=torch.float32)
    grouped_mm_mxfp4(a, part, s, offs, out=wide[:, 3:48])
    again = grouped_mm_mxfp4(a.contiguous(), part.contiguous(), s.contiguous(), offs, out_dtype=torch.float32)
    assert torch.equal(wide[:, 3:48], again) and not wide[:, :3].any() and not wide[:, 48:].any()
    assert torch.equal(matmul_mxfp4(a[:1].expand(5, 320), part[0], s[0]), matmul_mxfp4(a[:1].repeat(5, 1), part[0], s[0]))
    assert torch.equal(matmul_mxfp4(a[::3], part[0], s[0]), matmul_mxfp4(a[::3].contiguous(), part[0], s[0]))
    if hasattr(torch, "float4_e2m1fn_x2") and hasattr(torch, "float8_e8m0fnu"):
        typed = matmul_mxfp4(a, q[0, :, :160].view(torch.float4_e2m1fn_x2), scale[0, :, :10].view(torch.float8_e8m0fnu))
        assert torch.equal(typed, matmul_mxfp4(a, q[0, :, :160], scale[0, :, :10]))
    empty = matmul_mxfp4(a[:0], part[0], s[0])
    assert empty.shape == (0, 45)


def test_weights_past_four_gib():
    from kernels import grouped_mm_mxfp4

    groups, n, k = 40, 8192, 32768  # 5.4 GB of codes
    q = torch.randint(0, 256, (groups, n, k // 2), device="cuda", dtype=torch.uint8)
    scale = torch.randint(115, 120, (groups, n, k // 32), device="cuda", dtype=torch.uint8)
    a = normal(1, 3, k).to(torch.bfloat16)
    offs = torch.zeros(groups, device="cuda", dtype=torch.int32)
    offs[20:], offs[-1] = 1, 3
    out = grouped_mm_mxfp4(a, q, scale, offs)
    for part, e in ((slice(0, 1), 20), (slice(1, 3), groups - 1)):
        for cols in (slice(0, 64), slice(n - 64, n)):
            close(out[part, cols], a[part], values(q[e, cols], scale[e, cols]))


def test_calls_on_another_stream_and_in_a_replayed_graph():
    from kernels import dequantize_mxfp4, grouped_mm_mxfp4, grouped_mm_mxfp4_swiglu, quantize_mxfp4

    counts = [5, 0, 9, 1]
    offs = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    a, w13, w2 = normal(1, 15, 96).to(torch.bfloat16), normal(2, 4, 128, 96), normal(3, 4, 96, 64)

    def step():
        q13, q2 = quantize_mxfp4(w13), quantize_mxfp4(w2)
        h = grouped_mm_mxfp4_swiglu(a, *q13, offs)
        return (*q13, *q2, h, grouped_mm_mxfp4(h, *q2, offs), dequantize_mxfp4(*q2))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        there = step()
    torch.cuda.current_stream().wait_stream(stream)
    for x, y in zip(there, step()):
        assert torch.equal(x, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (7, 8, 9):
        a.copy_(normal(seed, 15, 96))
        w2.copy_(normal(seed + 1, 4, 96, 64))
        offs.copy_(torch.tensor([seed - 5, seed - 5, seed, 15], device="cuda"))
        expected = step()
        torch.cuda.synchronize()
        graph.replay()
        for x, y in zip(captured, expected):
            assert torch.equal(x, y)


def test_an_expert_layer_from_tokens_to_tokens():
    """Router, sort, gather, 4-bit experts and the weighted way back, as a decode step runs them, against 64 bits on the
    chosen experts.  h is rounded to bf16 between the products: 2^-8 of it, and the products' own bounds, come to less than
    2^-6 of the sum of sizes."""
    from kernels import (combine_rows, gather_rows, grouped_mm_mxfp4, grouped_mm_mxfp4_swiglu, quantize_mxfp4, route_topk,
                         sort_by_expert)

    tokens, experts, k, hidden, ffn = 37, 16, 4, 160, 96
    x = normal(1, tokens, hidden).to(torch.bfloat16)
    w13 = quantize_mxfp4(normal(2, experts, 2 * ffn, hidden) / hidden ** 0.5)
    w2 = quantize_mxfp4(normal(3, experts, hidden, ffn) / ffn ** 0.5)
    weights, chosen = route_topk(normal(4, tokens, experts), k)
    order = sort_by_expert(chosen, experts)
    h = grouped_mm_mxfp4_swiglu(gather_rows(x, order), *w13, order.offs)
    out = combine_rows(grouped_mm_mxfp4(h, *w2, order.offs), order, weights)
    v13, v2 = values(*w13), values(*w2)
    for t in range(tokens):
        exact = size = 0
        for j in range(k):
            e = int(chosen[t, j])
            p = v13[e] @ x[t].double()
            act = p[:ffn] * torch.sigmoid(p[:ffn]) * p[ffn:]
            exact = exact + float(weights[t, j]) * (v2[e] @ act)
            size = size + float(weights[t, j]) * (v2[e].abs() @ act.abs())
        assert bool(((out[t].double() - exact).abs() <= 2.0 ** -6 * size).all())
