"""GPU tests of the block-scaled fp8 operators against their definitions in 64 bits.

Bounds (derived, elementwise).  Products: e4m3 products are exact, so an output differs from the 64-bit
sum by at most the fp32 sums' rounding, (K + 8) 2^-23 sum_k |a w| (a unit of 2^-23 covers truncating adds),
plus half a unit of the output type.  With fast_accum the matrix instructions add eight products at a time and drop
what is below 2^-13 of the largest of them (FAST below): at most 8 x 2^-13 max over each eight, so 2^-10
sum_k |a w| in all.  Quantised values: half an e4m3 step is 2^-4 of a normal value and 2^-10 of the
scale below the normal range.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
HALF_UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.fixture(autouse=True)
def _gpu_only():
    if not torch.cuda.is_available():
        pytest.skip("ROCm GPU unavailable")


def normal(seed, *shape):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def blocked_amax(x, block_rows):
    """amax per block of a 2-D float64 tensor, with the definition's floor."""
    rows, k = x.shape
    padded = torch.zeros((-(-rows // block_rows) * block_rows, -(-k // 128) * 128), dtype=x.dtype, device=x.device)
    padded[:rows, :k] = x.abs()
    return padded.view(-1, block_rows, padded.shape[1] // 128, 128).amax(dim=(1, 3)).clamp(min=2.0 ** -96)


def spread(scale, block_rows, rows, k):
    return scale.double().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :k]


def operands(seed, rows, n, k, groups=None):
    """Quantised operands on 16-byte rows, made with torch, and their 64-bit values."""
    def quantised(x, block_rows):
        amax = blocked_amax(x.double(), block_rows)
        wide = spread(amax, block_rows, *x.shape)
        pitch = -(-x.shape[1] // 16) * 16
        buffer = torch.full((x.shape[0], pitch), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3)  # NaN in the padding
        q = buffer[:, :x.shape[1]]
        q.copy_((x.double() / wide * 448.0).float().to(E4M3))
        return buffer, (amax / 448.0).float()

    a, sa = quantised(normal(seed, rows, k) * normal(seed + 1, k).exp(), 1)
    weights = [quantised(normal(seed + 2 + e, n, k) / k ** 0.5 * normal(seed + 99, n, 1).exp(), 128)
               for e in range(groups or 1)]
    w = torch.stack([q for q, _ in weights])[:, :, :k] if groups else weights[0][0][:, :k]
    sw = torch.stack([s for _, s in weights]) if groups else weights[0][1]
    return a[:, :k], sa, w, sw


def values(q, scale, block_rows):
    return q.float().double() * spread(scale, block_rows, *q.shape)


FAST = 2.0 ** -10


def assert_product(out, a, sa, w, sw, more=0.0):
    """``out`` against a @ w.T of one group, elementwise; ``more``: further error per sum of |a w|."""
    x, y = values(a, sa, 1), values(w, sw, 128)
    exact, size = x @ y.t(), x.abs() @ y.abs().t()
    bound = HALF_UNIT[out.dtype] * exact.abs() + ((a.shape[1] + 8) * 2.0 ** -23 + more) * size + 2.0 ** -24
    worst = ((out.double() - exact).abs() - bound).max() if out.numel() else torch.tensor(-1.0)
    assert torch.isfinite(out).all() and float(worst) <= 0, float(worst)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 128), (3, 129), (17, 2880), (130, 1000), (300, 77), (128, 4096)])
def test_quantize_matches_the_definition(block_rows, dtype, rows, k):
    from kernels import quantize_fp8

    x = (normal(rows + k, rows, k) * normal(7, k).exp()).to(dtype)
    x[0, : min(k, 128)] = 0  # a run of zeros
    q, scale = quantize_fp8(x, block_rows=block_rows)
    amax = blocked_amax(x.double(), block_rows)
    torch.testing.assert_close(scale.double(), amax / 448.0, rtol=2.0 ** -23, atol=0)
    # The definition's own fp32 steps, on the CPU, give the same values bit for bit.
    inverse = (torch.tensor(448.0) / amax.float().cpu())
    wide = inverse.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :k]
    expected = (x.float().cpu() * wide).to(E4M3)
    assert torch.equal(q.cpu().contiguous().view(torch.uint8), expected.view(torch.uint8))
    error = (values(q, scale, block_rows) - x.double()).abs()
    step = spread(scale, block_rows, rows, k)
    assert bool((error <= 2.0 ** -4 * (1 + 2.0 ** -20) * x.double().abs() + 2.0 ** -10 * step).all())


def test_quantize_strides_batches_and_alignment():
    from kernels import quantize_fp8

    base = normal(3, 5, 70, 901).to(torch.bfloat16)
    for view in (base[:, 3:, 1:700], base[::2, ::3], base[:, :1], base[4]):  # odd offsets, strides, one row, 2-D
        for block_rows in (1, 128):
            q, scale = quantize_fp8(view, block_rows=block_rows)
            q0, scale0 = quantize_fp8(view.contiguous(), block_rows=block_rows)
            assert torch.equal(q.float(), q0.float()) and torch.equal(scale, scale0)
            assert q.stride(-2) % 16 == 0
    q, scale = quantize_fp8(base[0, :0])
    assert q.shape == (0, 901) and scale.shape == (0, 8)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_quantize_keeps_nan_and_infinity_in_their_block(bad):
    from kernels import quantize_fp8

    x = normal(5, 256, 384)
    clean = quantize_fp8(x, block_rows=128)
    x[130, 200] = bad
    q, scale = quantize_fp8(x, block_rows=128)
    value = q.float() * scale.repeat_interleave(128, 0).repeat_interleave(128, 1)
    assert torch.isnan(value[128:, 128:256]).all()
    assert torch.equal(q[:128].float(), clean[0][:128].float()) and torch.equal(scale[0], clean[1][0])
    q, scale = quantize_fp8(x)
    value = q.float() * scale.repeat_interleave(128, 1)
    assert torch.isnan(value[130, 128:256]).all() and int(torch.isnan(value).sum()) == 128


def test_quantize_tiny_and_huge_values():
    from kernels import quantize_fp8

    for factor in (2.0 ** -120, 2.0 ** -96, 2.0 ** 120):
        x = normal(9, 4, 256) * factor
        q, scale = quantize_fp8(x)
        assert torch.isfinite(q.float()).all() and torch.isfinite(scale).all()
        error = (q.float().double() * scale.double().repeat_interleave(128, 1) - x.double()).abs()
        assert bool((error <= 2.0 ** -4 * (1 + 2.0 ** -20) * x.double().abs()
                     + 2.0 ** -10 * scale.double().repeat_interleave(128, 1)).all())


def _variants(gated, fast=0):
    from kernels import _native

    lib = _native.library()
    return [v for v in range(lib.moegemm_fp8_variant_count(gated)) if lib.moegemm_fp8_variant_fast(gated, v) == fast]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 4096, 7168), (5, 72, 144), (16, 130, 2880), (33, 257, 1001),
                                   (70, 640, 129), (200, 264, 383), (513, 1032, 512)])
def test_matmul_matches_64_bits(m, n, k, dtype):
    from kernels import matmul_fp8

    a, sa, w, sw = operands(m + n + k, m, n, k)
    print(f"matmul_fp8 m={m} n={n} k={k} {dtype}", flush=True)
    out = matmul_fp8(a, sa, w, sw, out_dtype=dtype)
    assert out.dtype == dtype
    assert_product(out, a, sa, w, sw)


@pytest.mark.parametrize("m,n,k", [(1, 40, 16), (19, 300, 257), (260, 520, 400)])
def test_every_variant_matches_64_bits(m, n, k):
    from kernels import matmul_fp8

    a, sa, w, sw = operands(m * n + k, m, n, k)
    for variant in _variants(0):
        print(f"matmul_fp8 variant={variant} m={m} n={n} k={k}", flush=True)
        assert_product(matmul_fp8(a, sa, w, sw, variant=variant), a, sa, w, sw)
        again = matmul_fp8(a, sa, w, sw, variant=variant)
        assert torch.equal(again, matmul_fp8(a, sa, w, sw, variant=variant))


@pytest.mark.parametrize("counts,n,k", [((0, 3, 0, 16, 1), 136, 272), ((40, 0, 300, 17), 264, 640),
                                        ((1,) * 70, 64, 128), ((500, 100, 0, 29), 520, 260),
                                        ((0, 0, 0), 64, 128)])
def test_grouped_matches_64_bits(counts, n, k):
    from kernels import grouped_mm_fp8

    rows = sum(counts)
    offs = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    a, sa, w, sw = operands(rows + n, max(rows, 1), n, k, len(counts))
    a, sa = a[:rows], sa[:rows]
    for variant in (None, *_variants(0)):
        print(f"grouped_mm_fp8 counts={counts[:8]} n={n} k={k} variant={variant}", flush=True)
        out = grouped_mm_fp8(a, sa, w, sw, offs, variant=variant)
        assert out.shape == (rows, n)
        first = 0
        for e, count in enumerate(counts):
            part = slice(first, first + count)
            if count:
                assert_product(out[part], a[part], sa[part], w[e], sw[e])
            first += count


@pytest.mark.parametrize("counts,n,k", [((1,), 40, 16), ((40, 0, 300, 17), 264, 640), ((500, 100, 0, 29), 520, 260),
                                        ((700,), 1032, 1001)])
def test_fast_sums_stay_within_their_bound(counts, n, k):
    from kernels import grouped_mm_fp8

    rows = sum(counts)
    offs = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    a, sa, w, sw = operands(rows + n + 1, rows, n, k, len(counts))
    for variant in (None, *_variants(0, fast=1)):
        for dtype in (torch.bfloat16, torch.float32):
            print(f"fast grouped_mm_fp8 counts={counts} n={n} k={k} variant={variant} {dtype}", flush=True)
            out = grouped_mm_fp8(a, sa, w, sw, offs, fast_accum=True, variant=variant, out_dtype=dtype)
            first = 0
            for e, count in enumerate(counts):
                part = slice(first, first + count)
                first += count
                if count:
                    assert_product(out[part], a[part], sa[part], w[e], sw[e], FAST)


def test_rows_past_the_groups_stay_and_offsets_are_clamped():
    from kernels import grouped_mm_fp8

    a, sa, w, sw = operands(1, 90, 72, 160, 3)
    for variant in _variants(0):
        out = torch.full((90, 72), 7.0, device="cuda", dtype=torch.bfloat16)
        grouped_mm_fp8(a, sa, w, sw, torch.tensor([20, 20, 60], dtype=torch.int32, device="cuda"), out=out,
                       variant=variant)
        assert bool((out[60:] == 7.0).all())
        assert_product(out[:20], a[:20], sa[:20], w[0], sw[0])
        assert_product(out[20:60], a[20:60], sa[20:60], w[2], sw[2])
        grouped_mm_fp8(a, sa, w, sw, torch.tensor([-5, 30, 1000], dtype=torch.int32, device="cuda"), out=out,
                       variant=variant)
        assert_product(out[:30], a[:30], sa[:30], w[1], sw[1])
        assert_product(out[30:], a[30:], sa[30:], w[2], sw[2])


def test_strided_operands_scales_and_output():
    from kernels import matmul_fp8

    a, sa, w, sw = operands(11, 150, 200, 320)
    expected = matmul_fp8(a, sa, w, sw)
    wide = torch.zeros((300, 640), dtype=torch.uint8, device="cuda").view(E4M3)
    strided = wide[::2, 16:336]
    strided.copy_(a)
    scales = torch.zeros((300, 9), device="cuda")[::2, 1:4]
    scales.copy_(sa)
    out = torch.zeros((150, 403), device="cuda", dtype=torch.bfloat16)[:, 3:203]  # rows of odd alignment
    for scale in (scales, sa.t().contiguous().t(), sa[:1].expand(150, 3)):
        for variant in _variants(0):
            reference = expected if scale is not sa and scale.stride(0) else None
            got = matmul_fp8(strided, scale, w, sw.t().contiguous().t(), out=out, variant=variant)
            assert got is out
            if reference is not None:
                assert_product(out, a, sa, w, sw)
            else:
                assert_product(out, a, scale, w, sw)


def assert_quantised(q, scale, gate, up, gate_error, up_error):
    """(q, scale) against silu(gate) * up in 64 bits; the errors bound the fp32 gate and up."""
    h = gate * torch.sigmoid(gate) * up
    error = 1.1 * up.abs() * gate_error + (gate * torch.sigmoid(gate)).abs() * up_error + 1.1 * gate_error * up_error
    error = error + 2.0 ** -20 * h.abs()  # exp, reciprocal and the products
    rows, f = h.shape
    amax = blocked_amax(h, 1)
    slack = blocked_amax(error, 1) + 2.0 ** -22 * amax
    assert bool(((scale.double() * 448.0 - amax).abs() <= slack).all())
    step = spread(scale, 1, rows, f)
    difference = (q.float().double() * step - h).abs()
    assert bool((difference <= 2.0 ** -4 * (h.abs() + error) + 2.0 ** -10 * step + 2 * error).all())


@pytest.mark.parametrize("counts,f,k", [((3, 0, 1), 128, 256), ((1,), 8, 16), ((16, 40, 0, 7), 200, 400),
                                        ((150, 1, 0, 300), 264, 272), ((5, 33), 768, 2048), ((2, 600), 136, 130)])
def test_gated_matches_64_bits(counts, f, k):
    from kernels import grouped_mm_fp8_swiglu

    rows = sum(counts)
    offs = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    a, sa, w, sw = operands(rows + f, rows, 2 * f, k, len(counts))
    for fast, variant in ((0, None), (1, None), *((0, v) for v in _variants(1)), *((1, v) for v in _variants(1, 1))):
        print(f"grouped_mm_fp8_swiglu counts={counts} f={f} k={k} fast={fast} variant={variant}", flush=True)
        q, scale = grouped_mm_fp8_swiglu(a, sa, w, sw, offs, fast_accum=bool(fast), variant=variant)
        assert q.shape == (rows, f) and scale.shape == (rows, -(-f // 128)) and q.stride(0) % 16 == 0
        first = 0
        for e, count in enumerate(counts):
            part = slice(first, first + count)
            first += count
            if not count:
                continue
            x, y = values(a[part], sa[part], 1), values(w[e], sw[e], 128)
            p, size = x @ y.t(), ((k + 8) * 2.0 ** -23 + fast * FAST) * (x.abs() @ y.abs().t())
            assert_quantised(q[part], scale[part], p[:, :f], p[:, f:], size[:, :f], size[:, f:])


def test_one_group_without_offsets_and_the_chain_into_the_down_projection():
    from kernels import grouped_mm_fp8, grouped_mm_fp8_swiglu, matmul_fp8, quantize_fp8

    x = normal(21, 37, 512).to(torch.bfloat16)
    w13, w2 = normal(22, 400, 512) / 512 ** 0.5, normal(23, 96, 200) / 200 ** 0.5
    q, s = quantize_fp8(x)
    wq, ws = quantize_fp8(w13, block_rows=128)
    vq, vs = quantize_fp8(w2, block_rows=128)
    h, hs = grouped_mm_fp8_swiglu(q, s, wq, ws)
    offs = torch.tensor([37], dtype=torch.int32, device="cuda")
    h1, hs1 = grouped_mm_fp8_swiglu(q, s, wq[None], ws[None], offs)
    assert torch.equal(h.float(), h1.float()) and torch.equal(hs, hs1)
    y = matmul_fp8(h, hs, vq, vs, out_dtype=torch.float32)
    assert_product(y, h, hs, vq, vs)
    assert torch.equal(y, grouped_mm_fp8(h, hs, vq[None], vs[None], offs, out_dtype=torch.float32))
    # Against the unquantised layer: three roundings to 4 significant bits of independent values.
    p = x.double() @ w13.double().t()
    exact = (p[:, :200] * torch.sigmoid(p[:, :200]) * p[:, 200:]) @ w2.double().t()
    assert float((y.double() - exact).norm() / exact.norm()) < 2.0 ** -3


def test_graph_replays_read_new_offsets_and_other_streams_work():
    from kernels import grouped_mm_fp8, grouped_mm_fp8_swiglu

    a, sa, w, sw = operands(31, 64, 256, 256, 4)
    offs = torch.tensor([10, 20, 30, 64], dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        grouped_mm_fp8(a, sa, w, sw, offs)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = grouped_mm_fp8(a, sa, w, sw, offs)
        q, scale = grouped_mm_fp8_swiglu(a, sa, w, sw, offs)
    for ends in ([10, 20, 30, 64], [0, 0, 64, 64], [33, 40, 41, 64]):
        offs.copy_(torch.tensor(ends, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, grouped_mm_fp8(a, sa, w, sw, offs))
        eager = grouped_mm_fp8_swiglu(a, sa, w, sw, offs)
        assert torch.equal(q.float(), eager[0].float()) and torch.equal(scale, eager[1])


def test_nan_and_infinite_scales_reach_only_their_outputs():
    from kernels import matmul_fp8

    for m in (5, 300):
        a, sa, w, sw = operands(41, m, 300, 384)
        sa[2, 1] = float("nan")
        sw[1, 2] = float("inf")
        out = matmul_fp8(a, sa, w, sw)
        assert torch.isnan(out[2]).all()
        keep = [r for r in range(m) if r != 2]
        assert not torch.isfinite(out[keep, 128:256]).any()
        assert_product(out[keep][:, :128].contiguous(), a[keep], sa[keep], w[:128], sw[:1])


def test_offsets_past_32_bits():
    """Operands over 4 GiB: rows of a and experts of weight beyond 32-bit byte offsets."""
    from kernels import grouped_mm_fp8

    rows, k, n, groups = 300_000, 16384, 64, 2
    a = torch.zeros((rows, k), dtype=torch.uint8, device="cuda").view(E4M3)  # 4.9 GB
    a[-40:] = normal(51, 40, k).to(E4M3)
    w = normal(52, groups, n, k).to(E4M3)
    sa, sw = torch.ones((k // 128, rows), device="cuda").t(), torch.ones((groups, 1, k // 128), device="cuda")
    offs = torch.tensor([rows - 40, rows], dtype=torch.int32, device="cuda")
    out = grouped_mm_fp8(a, sa, w, sw, offs)
    assert not out[:-40].any()
    assert_product(out[-40:], a[-40:], sa[-40:], w[1], sw[1])


def test_more_groups_than_a_launch_lists():
    """Over 768 groups: several launches; groups of 0 to 2 rows, checked row by row."""
    from kernels import grouped_mm_fp8

    counts = [(i * 7) % 3 for i in range(1100)]
    rows, n, k = sum(counts), 40, 144
    offs = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    a, sa, w, sw = operands(3, rows, n, k, len(counts))
    owner = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), torch.tensor(counts, device="cuda"))
    x = values(a, sa, 1)
    y = torch.stack([values(w[e], sw[e], 128) for e in range(len(counts))])[owner]
    exact, size = (x[:, None] * y).sum(-1), (x[:, None] * y).abs().sum(-1)
    for variant in (None, *_variants(0)):
        print(f"grouped_mm_fp8 1100 groups variant={variant}", flush=True)
        out = grouped_mm_fp8(a, sa, w, sw, offs, variant=variant)
        bound = HALF_UNIT[out.dtype] * exact.abs() + (k + 8) * 2.0 ** -23 * size + 2.0 ** -24
        assert torch.isfinite(out).all() and ((out.double() - exact).abs() <= bound).all()


def test_more_rounds_than_a_launch_lists(monkeypatch):
    """300 tiles and more on one workgroup: the launches after the first start where it ended."""
    from kernels import fp8

    a, sa, w, sw = operands(4, 130, 128 * 300, 32)
    wide = fp8.matmul_fp8(a, sa, w, sw)
    monkeypatch.setattr(fp8, "_cu_count", lambda *_: 1)
    for variant in _variants(0):
        print(f"matmul_fp8 one workgroup variant={variant}", flush=True)
        out = fp8.matmul_fp8(a, sa, w, sw, variant=variant)
        assert_product(out[:, -640:], a, sa, w[-640:], sw[-5:])
        torch.testing.assert_close(out.float(), wide.float(), rtol=2.0 ** -7, atol=2.0 ** -7)


def test_quantize_more_rows_than_one_launch_takes():
    """2^28 rows and more are 2^24 workgroups of 256 threads: past the 2^32 threads of one launch."""
    from kernels import quantize_fp8

    rows, k = (1 << 28) + 37, 16
    x = torch.zeros((rows, k), device="cuda", dtype=torch.bfloat16)  # 8.6 GB
    middle = slice((1 << 27) - 5, (1 << 27) + 60)
    for part in (middle, slice(rows - 50, rows)):
        x[part] = normal(73, x[part].shape[0], k).to(torch.bfloat16)
    out = torch.full((rows, k), 0x7f, device="cuda", dtype=torch.uint8).view(E4M3)
    q, scale = quantize_fp8(x, out=out)
    for part in (middle, slice(rows - 50, rows)):
        expected = quantize_fp8(x[part].clone())
        assert torch.equal(q[part].float(), expected[0].float()) and torch.equal(scale[part], expected[1])
    for part in (slice(0, middle.start), slice(middle.stop, rows - 50)):
        assert not q[part].view(torch.uint8).any() and bool((scale[part] == 2.0 ** -96 / 448).all())


def test_more_rounds_than_a_launch_lists_with_fast_sums(monkeypatch):
    """The fast tiles over 300 tiles and more on one workgroup."""
    from kernels import fp8

    a, sa, w, sw = operands(4, 130, 128 * 300, 32)
    monkeypatch.setattr(fp8, "_cu_count", lambda *_: 1)
    for variant in _variants(0, fast=1):
        print(f"matmul_fp8 one workgroup, fast, variant={variant}", flush=True)
        out = torch.full((130, 128 * 300), float("nan"), device="cuda", dtype=torch.bfloat16)
        fp8.matmul_fp8(a, sa, w, sw, out=out, fast_accum=True, variant=variant)
        assert_product(out, a, sa, w, sw, FAST)


@pytest.mark.parametrize("cus", [1, 3])
@pytest.mark.parametrize("n,k", [(520, 80), (520, 144), (264, 400), (1032, 640)])
def test_several_tiles_a_workgroup(cus, n, k, monkeypatch):
    """A workgroup's stream of slices runs on over tiles of other groups and columns, one to five slices each."""
    from kernels import fp8

    counts = (130, 0, 300, 1, 64)
    rows = sum(counts)
    offs = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    a, sa, w, sw = operands(61 + n + k, rows, n, k, len(counts))
    monkeypatch.setattr(fp8, "_cu_count", lambda *_: cus)
    for fast in (0, 1):
        for variant in _variants(0, fast):
            for dtype in (torch.bfloat16, torch.float32):
                print(f"grouped_mm_fp8 cus={cus} n={n} k={k} fast={fast} variant={variant} {dtype}", flush=True)
                out = torch.full((rows, n), float("nan"), device="cuda", dtype=dtype)
                fp8.grouped_mm_fp8(a, sa, w, sw, offs, out=out, fast_accum=bool(fast), variant=variant)
                first = 0
                for e, count in enumerate(counts):
                    part = slice(first, first + count)
                    first += count
                    if count:
                        assert_product(out[part], a[part], sa[part], w[e], sw[e], fast * FAST)


@pytest.mark.parametrize("cus", [1, 2])
@pytest.mark.parametrize("f,k", [(200, 80), (264, 272), (392, 640)])
def test_several_gated_tiles_a_workgroup(cus, f, k, monkeypatch):
    """Gate and up rows, their scales and the row maxima change from tile to tile of one workgroup's stream."""
    from kernels import fp8

    counts = (40, 0, 150, 300, 1)
    rows = sum(counts)
    offs = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    a, sa, w, sw = operands(67 + f + k, rows, 2 * f, k, len(counts))
    monkeypatch.setattr(fp8, "_cu_count", lambda *_: cus)
    for fast, variant in (*((0, v) for v in _variants(1)), *((1, v) for v in _variants(1, 1))):
        print(f"grouped_mm_fp8_swiglu cus={cus} f={f} k={k} fast={fast} variant={variant}", flush=True)
        torch.full((rows, -(-f // 16) * 16), 0x7f, device="cuda", dtype=torch.uint8)  # NaN where nothing is written
        torch.full((-(-f // 128), rows), float("nan"), device="cuda")
        q, scale = fp8.grouped_mm_fp8_swiglu(a, sa, w, sw, offs, fast_accum=bool(fast), variant=variant)
        first = 0
        for e, count in enumerate(counts):
            part = slice(first, first + count)
            first += count
            if not count:
                continue
            x, y = values(a[part], sa[part], 1), values(w[e], sw[e], 128)
            p, size = x @ y.t(), ((k + 8) * 2.0 ** -23 + fast * FAST) * (x.abs() @ y.abs().t())
            assert_quantised(q[part], scale[part], p[:, :f], p[:, f:], size[:, :f], size[:, f:])


def test_rows_far_apart_pass_32_bits():
    """Rows of a and of the weight 8 MB apart: every kernel, streams too, past 4 GiB."""
    from kernels import grouped_mm_fp8, grouped_mm_fp8_swiglu

    rows, n, k, pitch = 600, 592, 256, (1 << 23) - 16
    a, sa, w, sw = operands(71, rows, n, k, 1)
    wide = torch.zeros((rows, pitch), dtype=torch.uint8, device="cuda").view(E4M3)  # 5.0 GB
    far_a, far_w = wide[:, :k], wide[None, :n, 512:512 + k]
    far_a.copy_(a), far_w.copy_(w)
    offs = torch.tensor([rows], dtype=torch.int32, device="cuda")
    for fast in (0, 1):
        for variant in _variants(0, fast):
            print(f"grouped_mm_fp8 rows 8 MB apart fast={fast} variant={variant}", flush=True)
            out = grouped_mm_fp8(far_a, sa, far_w, sw, offs, fast_accum=bool(fast), variant=variant)
            assert_product(out, a, sa, w[0], sw[0], fast * FAST)
        for variant in _variants(1, fast):
            print(f"grouped_mm_fp8_swiglu rows 8 MB apart fast={fast} variant={variant}", flush=True)
            q, scale = grouped_mm_fp8_swiglu(far_a, sa, far_w, sw, offs, fast_accum=bool(fast), variant=variant)
            near = grouped_mm_fp8_swiglu(a, sa, w, sw, offs, fast_accum=bool(fast), variant=variant)
            assert torch.equal(q.float(), near[0].float()) and torch.equal(scale, near[1])


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(37, 300), (3, 150, 264), (2, 1, 129)])
def test_quantize_into_given_buffers(shape, dtype, block_rows):
    """``out`` and ``scale`` of any layout get what a call without them returns, batches what each matrix alone gets, and
    nothing is written beside them."""
    from kernels import quantize_fp8

    x = normal(81, *shape).to(dtype)
    q, scale = quantize_fp8(x, block_rows=block_rows)
    *batch, rows, k = shape
    wide = torch.full((*batch, rows + 2, k // 8 * 8 + 40), 0x55, device="cuda", dtype=torch.uint8)
    out = wide[..., 1:rows + 1, 16:16 + k].view(E4M3)
    blocks = scale.shape[-2:]
    for given in (torch.full((*batch, *blocks), -1.0, device="cuda"),
                  torch.full((*batch, blocks[1], blocks[0] + 3), -1.0, device="cuda")[..., 2:2 + blocks[0]].transpose(-1, -2),
                  torch.full((*batch, 2 * blocks[0], 3 * blocks[1]), -1.0, device="cuda")[..., ::2, 1::3]):
        got = quantize_fp8(x, block_rows=block_rows, out=out, scale=given)
        assert got[0] is out and got[1] is given
        assert torch.equal(out.float(), q.float()) and torch.equal(given, scale)
        if given._base is not None:
            assert int((given._base != -1.0).sum()) == given.numel()
    untouched = torch.ones_like(wide, dtype=torch.bool)
    untouched[..., 1:rows + 1, 16:16 + k] = False
    assert bool((wide[untouched] == 0x55).all())
    if batch:
        for i in range(batch[0]):
            alone = quantize_fp8(x[i], block_rows=block_rows)
            assert torch.equal(alone[0].float(), q[i].float()) and torch.equal(alone[1], scale[i])


def test_refusals_of_given_buffers():
    from kernels import grouped_mm_fp8, matmul_fp8, quantize_fp8

    x = normal(83, 8, 256)
    e4m3 = torch.zeros((8, 300), dtype=torch.uint8, device="cuda").view(E4M3)
    for out in (e4m3, e4m3[:, 4:260], e4m3[:, :256].float(), e4m3[:, :256].cpu(), e4m3[:4, :256], e4m3[:1, :256].expand(8, 256)):
        with pytest.raises(ValueError, match="out must be"):
            quantize_fp8(x, out=out)
    for scale in (torch.zeros(8, 1, device="cuda"), torch.zeros(8, 2), torch.zeros(8, 2, device="cuda").double()):
        with pytest.raises(ValueError, match="scale must be"):
            quantize_fp8(x, scale=scale)
    with pytest.raises(ValueError, match="unit stride"):
        quantize_fp8(x.t())
    with pytest.raises(ValueError):
        quantize_fp8(x.int())
    a, sa, w, sw = operands(85, 8, 32, 256, 1)
    offs = torch.tensor([8], dtype=torch.int32, device="cuda")
    for out in (torch.zeros(8, 31, device="cuda"), torch.zeros(8, 32), torch.zeros(32, 8, device="cuda").t()):
        with pytest.raises(ValueError, match="out must be"):
            grouped_mm_fp8(a, sa, w, sw, offs, out=out)
    with pytest.raises(ValueError, match="out_dtype"):
        matmul_fp8(a, sa, w[0], sw[0], out=torch.zeros(8, 32, device="cuda"), out_dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="cover"):
        matmul_fp8(a, sa, w[0], sw[0], out=torch.zeros(1, 32, device="cuda").expand(8, 32))
    for bad in (offs.long(), torch.cat([offs, offs]), offs.cpu()):
        with pytest.raises(ValueError, match="offs|device"):
            grouped_mm_fp8(a, sa, w, sw, bad)
    with pytest.raises(ValueError, match="16 bytes"):
        matmul_fp8(e4m3[:, 8:264], sa, w[0], sw[0])


def test_strided_experts_and_scales():
    """Every other expert of a larger weight, and scales to match."""
    from kernels import grouped_mm_fp8, grouped_mm_fp8_swiglu

    counts = (5, 0, 70)
    offs = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    a, sa, w, sw = operands(87, 75, 64, 272, 3)
    more = torch.full((6, 128, 288), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3)
    far_w = more[::2, ::2, 16:288]
    far_w.copy_(w)
    far_sw = torch.full((6, 3, 7), float("nan"), device="cuda")[1::2, 1:2, ::3]
    far_sw.copy_(sw)
    assert torch.equal(grouped_mm_fp8(a, sa, far_w, far_sw, offs), grouped_mm_fp8(a, sa, w, sw, offs))
    one, other = grouped_mm_fp8_swiglu(a, sa, far_w, far_sw, offs), grouped_mm_fp8_swiglu(a, sa, w, sw, offs)
    assert torch.equal(one[0].float(), other[0].float()) and torch.equal(one[1], other[1])
    shared = w[:1].expand(3, 64, 272), sw[:1].expand(3, 1, 3)  # one weight for all
    alone = grouped_mm_fp8(a, sa, *shared, offs)
    for part in (slice(0, 5), slice(5, 75)):
        assert_product(alone[part], a[part], sa[part], w[0], sw[0])


def test_quantize_one_row_into_a_dense_buffer():
    """A single row starts where the buffer does, whatever its pitch; so does the only matrix of a batch of one."""
    from kernels import quantize_fp8

    for shape in ((1, 129), (1, 1, 77), (1, 3, 40)):
        x = normal(89, *shape)
        out = torch.zeros(shape, dtype=torch.uint8, device="cuda").view(E4M3)
        if shape == (1, 3, 40):
            out = torch.as_strided(out, shape, (123, 40, 1))
        for block_rows in (1, 128):
            expected = quantize_fp8(x, block_rows=block_rows)
            q, scale = quantize_fp8(x, block_rows=block_rows, out=out)
            assert q is out and torch.equal(q.float(), expected[0].float()) and torch.equal(scale, expected[1])
