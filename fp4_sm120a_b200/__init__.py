"""B200-native (sm_100a) NVFP4 quantization: the RHT GEMM + NVFP4 cast
(rht_gemm_ntt_w_sfc), the four FP4 stochastic-rounding conversions and the
scaled FP8 conversions of Harry-Chen/fp4_sm120a, and the training step around
the cast (products of NVFP4 operands, layer norm, AdamW), behind a C ABI
(include/nvfp4_b200.h)."""
from ._native import NVFP4Error, library_path, load  # noqa: F401
from .ops import (  # noqa: F401
    amax_bf16,
    amax_bf16_chained,
    adamw_step,
    cvt_fp32_to_fp4_4x_sr,
    device_error,
    gemm_nvfp4,
    gemm_nvfp4_dact,
    gemm_nvfp4_dact_workspace_bytes,
    gemm_nvfp4_workspace_bytes,
    hadamard16,
    layernorm_bwd,
    layernorm_bwd_workspace_bytes,
    layernorm_fwd,
    mul_cvt_bf16_to_fp4_4x_sr,
    mul_cvt_bf16_to_fp4_8x_sr,
    mul_cvt_fp32_to_fp4_4x_sr,
    mul_cvt_fp8_2x,
    mul_cvt_fp8_4x,
    quantize_rht,
    quantize_rht_fused,
    quantize_rht_fused_sharded_exchange,
    fused_workspace,
    quantize_rowwise_bf16_sr,
    rht_gemm_ntt_w_sfc,
    rht_gemm_ntt_w_sfc_sharded,
    rht_gemm_ntt_w_sfc_sharded_exchange,
    PeerExchange,
    rht_gemm_ttt_wrapper,
)
from .training import (  # noqa: F401
    AdamW,
    adamw_unpack_state,
    layernorm,
    layernorm_backward,
    matmul_nvfp4,
    matmul_nvfp4_dact,
)

__version__ = "0.1.0"
