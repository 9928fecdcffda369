"""gfx950 HIP grouped/single GEMM kernels, routing, and the PyTorch grouped_mm comparison provider."""

from .fp8 import grouped_mm_fp8, grouped_mm_fp8_swiglu, matmul_fp8, quantize_fp8
from .gated_ffn import gate_up_swiglu, gate_up_swiglu_backward, gate_up_swiglu_forward
from .grouped_gemm import (
    GroupedWorkspace,
    build_fused_gate_up_workspace,
    build_grouped_workspace,
    grouped_candidate_configs,
    launch_gate_up_swiglu,
    launch_grouped,
)
from .grouped_mm import (
    OffsetsWorkspace,
    build_offsets_workspace,
    grouped_mm,
    grouped_mm_swiglu,
    last_grouped_mm_config,
    last_grouped_mm_schedule,
    launch_grouped_offsets,
)
from .matmul import (
    KernelConfig,
    last_matmul_config,
    launch_matmul,
    matmul_candidate_configs,
    select_config,
)
from .mxfp4 import dequantize_mxfp4, grouped_mm_mxfp4, grouped_mm_mxfp4_swiglu, matmul_mxfp4, quantize_mxfp4
from .routing import (
    ExpertOrder,
    combine_rows,
    combine_rows_backward,
    gather_rows,
    route_topk,
    route_topk_backward,
    sort_by_expert,
)
from .torch_grouped_gemm import (
    TorchGroupedMMUnavailable,
    TorchGroupedWorkspace,
    build_torch_grouped_workspace,
    launch_torch_grouped,
    torch_grouped_mm_unavailable_reason,
)

__all__ = [
    "ExpertOrder",
    "GroupedWorkspace",
    "KernelConfig",
    "OffsetsWorkspace",
    "TorchGroupedMMUnavailable",
    "TorchGroupedWorkspace",
    "build_fused_gate_up_workspace",
    "build_grouped_workspace",
    "build_offsets_workspace",
    "build_torch_grouped_workspace",
    "combine_rows",
    "combine_rows_backward",
    "dequantize_mxfp4",
    "gate_up_swiglu",
    "gate_up_swiglu_backward",
    "gate_up_swiglu_forward",
    "gather_rows",
    "grouped_candidate_configs",
    "grouped_mm",
    "grouped_mm_fp8",
    "grouped_mm_fp8_swiglu",
    "grouped_mm_mxfp4",
    "grouped_mm_mxfp4_swiglu",
    "grouped_mm_swiglu",
    "last_grouped_mm_config",
    "last_grouped_mm_schedule",
    "last_matmul_config",
    "launch_gate_up_swiglu",
    "launch_grouped",
    "launch_grouped_offsets",
    "launch_matmul",
    "launch_torch_grouped",
    "matmul_candidate_configs",
    "matmul_fp8",
    "matmul_mxfp4",
    "quantize_fp8",
    "quantize_mxfp4",
    "route_topk",
    "route_topk_backward",
    "select_config",
    "sort_by_expert",
    "torch_grouped_mm_unavailable_reason",
]
