from .batch_gemm import batch_gemm
from .block_scale import block_gemm, block_quant, group_block_gemm, swiglu_block_quant
from .dense_gemm import EpilogueOp, dense_gemm, interleave_gate_up
from .group_gemm import group_contiguous_gemm, group_masked_gemm
from .group_wise_quant import group_wise_quant
from .low_latency_mma_gemm import low_latency_mma_gemm
from .rms_norm_quant import rms_norm_quant

__all__ = ["EpilogueOp", "batch_gemm", "block_gemm", "block_quant", "dense_gemm", "group_block_gemm", "group_contiguous_gemm", "group_masked_gemm",
           "group_wise_quant", "interleave_gate_up", "low_latency_mma_gemm", "rms_norm_quant", "swiglu_block_quant"]
