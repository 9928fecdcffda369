"""GPU tests of infinite values in the rows of 4-bit products, beside weights large enough to overflow what a split leaves."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
INF = float("inf")

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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("low,high", [(115, 126), (136, 137), (160, 201)])
def test_infinities_keep_their_sign_beside_large_weights(low, high, dtype):
    """Weights of 2^-12 to 2^74 in both signs: an infinite value gives an infinity of the product's sign, other rows what
    they give without it."""
    from kernels import matmul_mxfp4

    q, scale = random_weight(high, 50, 288, low, high)
    q |= 0x11  # no zeros, whose product with an infinity is no number
    w = values(q, scale)
    a = normal(4, 11, 288).to(dtype)
    for variant in variants():
        clean = matmul_mxfp4(a, q, scale, out_dtype=torch.float32, variant=variant)
        b = a.clone()
        b[3, 100], b[7, 287] = INF, -INF
        out = matmul_mxfp4(b, q, scale, out_dtype=torch.float32, variant=variant)
        assert torch.equal(out[3].double(), INF * w[:, 100]), variant
        assert torch.equal(out[7].double(), -INF * w[:, 287]), variant
        keep = [r for r in range(11) if r not in (3, 7)]
        assert torch.isfinite(out[keep]).all() and torch.equal(out[keep], clean[keep])
