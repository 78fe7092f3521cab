"""Operator wrappers with the signatures of ``nunchaku.ops`` (nunchaku/ops/{quantize,gemm,fused}.py), and the 8-bit linear
operators, attention, norms and rotary positions that stand beside them."""

from .attention import cross_attention, self_attention
from .fused import fused_gelu_mlp, fused_qkv_norm_rottary, linearattn_vk_mul_q
from .gemm import svdq_gemm_w4a4, svdq_gemm_w4a4_cuda
from .gemv import awq_gemv_w4a16, awq_gemv_w4a16_cuda
from .norm import gated_norm
from .quantize import svdq_quantize_w4a4_act_fuse_lora, svdq_quantize_w4a4_act_fuse_lora_cuda
from .rotary import rotary_axes
from .w8a8 import gemm_w8a8, quantize_w8a8_act, rms_norm_quantize_w8a8

__all__ = [
    "svdq_quantize_w4a4_act_fuse_lora",
    "svdq_quantize_w4a4_act_fuse_lora_cuda",
    "svdq_gemm_w4a4",
    "svdq_gemm_w4a4_cuda",
    "awq_gemv_w4a16",
    "awq_gemv_w4a16_cuda",
    "fused_gelu_mlp",
    "fused_qkv_norm_rottary",
    "linearattn_vk_mul_q",
    "quantize_w8a8_act",
    "rms_norm_quantize_w8a8",
    "gemm_w8a8",
    "cross_attention",
    "self_attention",
    "gated_norm",
    "rotary_axes",
]
