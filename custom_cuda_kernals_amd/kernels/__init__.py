"""Python entry points, one module per op, with the reference's signatures
(custom_cuda/kernels/{rmsnorm_residual,swiglu,rope,fp8_quant,token_permute,moe_router}.py)
plus the additive FP8 modes and fusions, the expert products, MXFP4, the
products of block-scaled FP8, and the decode step's ops (rotary positions, the paged
cache and its attention)."""

from custom_cuda_kernals_amd.kernels.fp8_linear import fp8_block_linear
from custom_cuda_kernals_amd.kernels.fp8_quant import fp8_quant
from custom_cuda_kernals_amd.kernels.grouped_linear import (
    grouped_linear,
    grouped_linear_grad_input,
    grouped_linear_grad_weight,
)
from custom_cuda_kernals_amd.kernels.moe_router import moe_router
from custom_cuda_kernals_amd.kernels.mxfp4 import mxfp4_dequant, mxfp4_linear, mxfp4_quant
from custom_cuda_kernals_amd.kernels.paged_attention import paged_attention, rope_to_cache
from custom_cuda_kernals_amd.kernels.rmsnorm_residual import rmsnorm_residual, rmsnorm_residual_fp8
from custom_cuda_kernals_amd.kernels.rope import rope
from custom_cuda_kernals_amd.kernels.rotary import rope_at, rope_frequencies
from custom_cuda_kernals_amd.kernels.swiglu import swiglu, swiglu_fp8
from custom_cuda_kernals_amd.kernels.token_permute import compute_permutation, token_combine, token_gather

__all__ = ["fp8_quant", "rmsnorm_residual", "rmsnorm_residual_fp8", "rope", "swiglu", "swiglu_fp8",
           "token_gather", "token_combine", "compute_permutation", "moe_router", "grouped_linear", "grouped_linear_grad_input",
           "grouped_linear_grad_weight", "mxfp4_quant", "mxfp4_dequant", "mxfp4_linear",
           "rope_at", "rope_frequencies", "rope_to_cache", "paged_attention", "fp8_block_linear"]
