"""GPU tests of what the 4-bit products make of fp32 rows, whose 24 bits they keep."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


@pytest.fixture(autouse=True)
def _gpu_only():
    if not torch.cuda.is_available():
        pytest.skip("ROCm GPU unavailable")


def normal(seed, *shape):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def variants():
    from kernels import _native

    return [None, *range(_native.library().moegemm_mxfp4_variant_count())]


def random_weight(seed, n, k, low, high):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 256, (n, k // 2), device="cuda", dtype=torch.uint8, generator=generator)
    return q, torch.randint(low, high, (n, k // 32), device="cuda", dtype=torch.uint8, generator=generator)


def values(q, scale):
    """64-bit values of packed bytes."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device=q.device)
    code = torch.stack([q & 15, q >> 4], dim=-1).reshape(*scale.shape, 32)
    return (table[code.long()] * torch.exp2(scale.double() - 127)[..., None]).reshape(*scale.shape[:-1], -1)


def fp32_patterns(seed, count, low, high):
    """Random sign and significand bits under exponent fields low to high - 1."""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    bits = torch.randint(0, 1 << 23, (count,), device="cuda", generator=generator)
    bits |= torch.randint(low, high, (count,), device="cuda", generator=generator) << 23
    sign = torch.randint(0, 2, (count,), device="cuda", generator=generator) << 31
    return (bits | sign).to(torch.int64).sub((sign > 0).long() << 32).to(torch.int32).view(torch.float32)


def test_fp32_rows_keep_all_their_bits():
    """Single products of 1: every fp32 value from 2^-110 up comes back whole.  Three bf16 parts hold its 24 bits, and their
    sums in order are exact.  Below, the last part is a multiple of 2^-133, rounded to it: off by 2^-134 at most."""
    from kernels import matmul_mxfp4

    q = torch.zeros(32, 16, dtype=torch.uint8, device="cuda")
    for i in range(32):
        q[i, i // 2] = 2 << (4 * (i % 2))  # 1.0 on the diagonal
    one = torch.full((32, 1), 127, dtype=torch.uint8, device="cuda")
    ends = torch.tensor([1.0, torch.finfo(torch.float32).max, -torch.finfo(torch.float32).max, 2.0 ** -110, 1 + 2.0 ** -23, 0.0])
    a = torch.cat([fp32_patterns(1, 32 * 500 - 6, 17, 255), ends.cuda()]).view(-1, 32)
    small = fp32_patterns(2, 32 * 60, 0, 17).view(-1, 32)
    for variant in variants():
        assert torch.equal(matmul_mxfp4(a, q, one, variant=variant), a), variant
        off = (matmul_mxfp4(small, q, one, variant=variant).double() - small.double()).abs()
        assert float(off.max()) <= 2.0 ** -134, variant


@pytest.mark.parametrize("m,n,k", [(1, 70, 2880), (4, 33, 64), (17, 100, 7168), (40, 64, 544), (70, 96, 256)])
def test_products_of_fp32_rows(m, n, k):
    """Rows of five values among zeros, so that few sums round: 15 parts' products, and 4 sums of waves and halves, each of
    2^-23 of sum |a w| at most; 2^-24 of the result."""
    from kernels import matmul_mxfp4

    a = torch.zeros(m, k, device="cuda")
    at = torch.rand(m, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(k)).topk(5, dim=1).indices
    a.scatter_(1, at, normal(m + n, m, 5))
    q, scale = random_weight(k, n, k, 115, 125)
    w = values(q, scale)
    exact, size = a.double() @ w.t(), a.double().abs() @ w.abs().t()
    for variant in variants():
        out = matmul_mxfp4(a, q, scale, variant=variant)
        assert out.dtype is torch.float32
        assert bool(((out.double() - exact).abs() <= 19 * 2.0 ** -23 * size + 2.0 ** -24 * exact.abs()).all()), variant
