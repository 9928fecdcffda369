"""harness.expert_layer's routed 4-bit experts against bf16 experts of the very values that the 4 bits stand for."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,top_k", [(1, 6), (3, 1), (60, 2), (400, 3)])
def test_routed_experts_of_equal_weights_agree(tokens, top_k):
    """Both round h, each expert's row and the token to bf16, 2^-8 each of sum_j weight |h| |w2|, and their fp32 sums by less
    than 2^-12 of it: (3 2^-8 + 2^-12) on either side, and a little for the roundings' product."""
    if not torch.cuda.is_available():
        pytest.skip("ROCm GPU unavailable")
    from harness.expert_layer import ExpertLayer, LayerSizes, Mxfp4ExpertLayer, routed
    from kernels import dequantize_mxfp4, route_topk

    experts, hidden, ffn = 6, 256, 160
    layer = ExpertLayer(LayerSizes(experts, hidden, ffn, 0, 0, top_k), torch.device("cuda"), 7)
    small = Mxfp4ExpertLayer(layer)
    layer.w13 = dequantize_mxfp4(*small.w13).transpose(1, 2).contiguous()
    layer.w2 = dequantize_mxfp4(*small.w2).transpose(1, 2).contiguous()
    generator = torch.Generator(device="cuda").manual_seed(tokens)
    x = torch.randn(tokens, hidden, device="cuda", generator=generator).bfloat16()
    logits = torch.randn(tokens, experts, device="cuda", generator=generator)
    ours, theirs = (routed(each, x, logits, top_k).double() for each in (small, layer))

    weights, chosen = route_topk(logits, top_k)
    exact = size = 0
    for e in range(experts):
        share = torch.where(chosen == e, weights, 0.0).double().sum(dim=1, keepdim=True)  # [T, 1]
        gate, up = (x.double() @ layer.w13[e].double()).chunk(2, dim=1)
        h, w2 = gate * torch.sigmoid(gate) * up, layer.w2[e].double()
        exact, size = exact + share * (h @ w2), size + share * (h.abs() @ w2.abs())
    bound = (3 * 2.0 ** -8 + 2.0 ** -12 + 2.0 ** -14) * size
    assert bool(((ours - exact).abs() <= bound).all()) and bool(((theirs - exact).abs() <= bound).all())
