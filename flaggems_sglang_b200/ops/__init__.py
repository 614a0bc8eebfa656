"""Operators of the fused-MoE path and of what stands beside it in a layer (flat namespace, no vendor registry)."""
from .fused_moe import (  # noqa: F401
    GatherIndx,
    RoutingData,
    ScatterIndx,
    fused_experts,
    fused_moe,
    fused_moe_flagos,
    standard_topk_to_routing,
    triton_kernel_fused_experts,
    triton_kernel_fused_experts_with_bias,
)
from .linear import fp8_block_linear, fp8_gated_mlp  # noqa: F401
from .moe_align_block_size import moe_align_block_size  # noqa: F401
from .moe_sum import moe_sum  # noqa: F401
from .norm import rms_norm_quant_fp8  # noqa: F401
from .quant import (  # noqa: F401
    per_token_group_quant_fp8, per_token_quant_fp8, quant_weight_block128, quant_weight_per_channel,
)
from .topk import fused_topk, grouped_topk, topk  # noqa: F401

__all__ = [
    "fused_experts", "fused_moe", "triton_kernel_fused_experts", "triton_kernel_fused_experts_with_bias",
    "fused_moe_flagos",
    "standard_topk_to_routing", "RoutingData", "GatherIndx", "ScatterIndx",
    "moe_align_block_size", "moe_sum", "per_token_group_quant_fp8", "quant_weight_block128",
    "per_token_quant_fp8", "quant_weight_per_channel",
    "rms_norm_quant_fp8", "fp8_block_linear", "fp8_gated_mlp",
    "fused_topk", "grouped_topk", "topk",
]
