"""Microscaled (MX) linears on MI355X: 4-bit floating-point weights, activations quantised to 8- or 4-bit floating point, one
power-of-two scale for every 32 consecutive values.  They stand beside the AWQ linears of `layers.gemm`: half a byte a weight
there and here, but here the products run in 8 or 4 bits on the matrix cores, several times the 16-bit rate.

`format` is "mxfp8" (elements e4m3) or "mxfp4" (e2m1, two a byte, the first in the low half).  Codes and scales are uint8,
`[..., k]` or `[..., k / 2]` and `[..., k / 32]`; a scale byte s is 2^(s - 127), and 255 stands for a block of NaN, which is
what a block with an infinity or a NaN becomes.  Scales are chosen so that every value is rounded to nearest and none
saturates.  k is a multiple of 32.  Weights are "mxfp4" rows `[out_features, in_features / 2]`.

Everything runs on HIP kernels behind `torch.ops.nanoquantization_amd.mx_*`, on the current stream of the tensors' device, and
has no derivative; there is no CPU path.  The reference has no counterpart (its linears multiply in 16 bits)."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from .. import _lib

MX_BLOCK = 32
MX_FORMATS = ("mxfp4", "mxfp8")


class _Operators:
    """torch.ops.nanoquantization_amd.mx_*, looked up once."""

    def __getattr__(self, name: str):
        op = getattr(_lib.mx_ops(), name).default
        setattr(self, name, op)
        return op


_ops = _Operators()


def _elsewhere(t: torch.Tensor):
    return _lib.AwqHipError("MX kernels run on a HIP device only (tensor is on %s); there is no CPU fallback" % t.device)


def mx_quantize(x: torch.Tensor, format: str = "mxfp4") -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of x [..., k], float16, bfloat16 or float32."""
    if not x.is_cuda:
        raise _elsewhere(x)
    return _ops.mx_quantize(x, format)


def mx_dequantize(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [..., k] that codes and scales stand for, rounded once to `dtype`; the format follows from the sizes."""
    if not codes.is_cuda:
        raise _elsewhere(codes)
    return _ops.mx_dequantize(codes, scales, dtype)


def mx_linear(x: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, bias: Optional[torch.Tensor] = None,
              activations: str = "mxfp8") -> torch.Tensor:
    """x [..., k] quantised to `activations`, times weight^T, plus bias: [..., n] in x's dtype.  Sums in fp32, one rounding
    behind the bias.  A bias of another dtype than x is rounded to x's first, by a launch of its own."""
    if not x.is_cuda:
        raise _elsewhere(x)
    return _ops.mx_linear(x, weight, weight_scales, bias, activations)


def mx_linear_quantized(codes: torch.Tensor, scales: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor,
                        bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The same product for activations that are quantised already (by mx_quantize, mx_add_rmsnorm or mx_silu_mul); `dtype` takes
    the place of x's."""
    if not codes.is_cuda:
        raise _elsewhere(codes)
    return _ops.mx_linear_quantized(codes, scales, weight, weight_scales, bias, dtype)


def mx_add_rmsnorm(x: torch.Tensor, delta: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6,
                   format: str = "mxfp8") -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(codes, scales, total): total = x + delta in x's dtype, and the quantised RMSNorm of it times `weight`, computed in fp32
    from the rounded sum.  Without a delta total is x itself.  At most 16384 values a row."""
    if not x.is_cuda:
        raise _elsewhere(x)
    if delta is None:
        codes, scales = _ops.mx_rmsnorm(x, weight, eps, format)
        return codes, scales, x
    return _ops.mx_add_rmsnorm(x, delta, weight, eps, format)


def mx_silu_mul(gate: torch.Tensor, up: torch.Tensor, format: str = "mxfp8") -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of SiLU(gate) * up, computed in fp32; the halves of one tensor [..., 2 k] are read in place."""
    if not gate.is_cuda:
        raise _elsewhere(gate)
    return _ops.mx_silu_mul(gate, up, format)


class MXLinear(nn.Module):
    """A linear of 4-bit floating-point weights.  `forward` takes a tensor, which is quantised to `activations` on the way, or
    (codes, scales) of one, as mx_add_rmsnorm and mx_silu_mul leave them; then the result is of `output_dtype`."""

    def __init__(self, in_features: int, out_features: int, bias: bool = False, activations: str = "mxfp8",
                 device: "str | torch.device" = "cpu", output_dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        if activations not in MX_FORMATS:
            raise ValueError(f"activations must be one of {MX_FORMATS}, got {activations!r}")
        assert in_features > 0 and in_features % MX_BLOCK == 0, "in_features must be a multiple of 32"
        self.in_features, self.out_features = in_features, out_features
        self.activations, self.output_dtype = activations, output_dtype
        self.register_buffer("weight", torch.zeros(out_features, in_features // 2, dtype=torch.uint8, device=device))
        self.register_buffer("weight_scales", torch.zeros(out_features, in_features // MX_BLOCK, dtype=torch.uint8, device=device))
        self.register_buffer("bias", torch.zeros(out_features, dtype=output_dtype, device=device) if bias else None)

    @classmethod
    def from_linear(cls, linear: nn.Linear, activations: str = "mxfp8",
                    output_dtype: Optional[torch.dtype] = None) -> "MXLinear":
        """Quantises the weight of a linear that lies on a HIP device.  `output_dtype` is that of its bias too; without one results
        of (codes, scales) are of the weight's dtype, or bfloat16 for a float32 weight, and the bias is held as the linear has it."""
        w = linear.weight.detach()
        made = cls(linear.in_features, linear.out_features, linear.bias is not None, activations, "meta",
                   output_dtype or (w.dtype if w.dtype != torch.float32 else torch.bfloat16))
        made.weight, made.weight_scales = mx_quantize(w, "mxfp4")
        if linear.bias is not None:
            made.bias = linear.bias.detach().to(output_dtype or linear.bias.dtype, copy=True)
        return made

    def forward(self, x) -> torch.Tensor:
        if isinstance(x, tuple):
            return mx_linear_quantized(*x, self.weight, self.weight_scales, self.bias, self.output_dtype)
        return mx_linear(x, self.weight, self.weight_scales, self.bias, self.activations)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, activations={self.activations}, "
                f"bias={self.bias is not None}")
