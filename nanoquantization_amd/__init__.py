"""MI355X (gfx950) native AWQ W4A16 linear path.

Host-side mirror of nanoquantization/layers/gemm.py and
nanoquantization/utils/quantization.py of liyuan24/nanoquantization, running on
hand-written HIP kernels (csrc/) behind the C ABI of include/awq_hip.h.
"""
from .layers.gemm import (WQLinear_GEMM, awq_dequantize, awq_dequantize_transposed, awq_gemm,  # noqa: F401
                          prefetch_hint)
from .layers.mx import (MXLinear, mx_add_rmsnorm, mx_dequantize, mx_linear, mx_linear_quantized, mx_quantize,  # noqa: F401
                        mx_silu_mul)
from .utils.quantization import pseudo_quantize, quantize_pack  # noqa: F401

__all__ = ["WQLinear_GEMM", "awq_dequantize", "awq_dequantize_transposed", "awq_gemm", "pseudo_quantize", "quantize_pack",
           "prefetch_hint", "MXLinear", "mx_add_rmsnorm", "mx_dequantize", "mx_linear", "mx_linear_quantized", "mx_quantize",
           "mx_silu_mul"]
