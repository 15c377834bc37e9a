/* C ABI of libnq_mx.so: microscaled (MX) formats -- quantising rows, the product of such rows with 4-bit weights, and the
 * steps of a decoder layer that leave their result in this form.
 *
 * A block of 32 consecutive values v of a row is held as one scale byte and 32 elements.  The scale is 2^e as the byte
 * e + 127; the elements are v / 2^e, rounded to nearest with ties to even, as
 *   NQX_FP4  e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two codes a byte, the first in the low half, or
 *   NQX_FP8  e4m3 (largest 448), one byte each.
 * e is the smallest exponent with which the block's largest magnitude, rounded to the nearest element, is not past the
 * largest element, and at least -127: no value is off by more than half a step.  A block with an infinity or a NaN has the
 * scale byte 255 and codes 0, and stands for NaN.  Magnitudes from 1.75 * 2^127 on may round up to 2^128, past fp32.
 * (Element and scale types are those of the OCP Microscaling Formats specification; its own scale, without the exponent's
 * step up, saturates the largest values and is off by more: normal values 0.115 instead of 0.112 in e2m1 and 0.0293 instead
 * of 0.0266 in e4m3, relative.)
 *
 * Layout: codes [rows, k / 2] (NQX_FP4) or [rows, k] (NQX_FP8), scales [rows, k / 32], both uint8 and dense row-major;
 * k % 32 == 0.  Weights are NQX_FP4, [n, k / 2] and [n, k / 32]: the rows of a torch Linear weight.
 *
 * Conventions: device pointers on the current HIP device, 16-byte aligned except scales and biases (any address of their
 * type).  `dtype` is the type of the unquantised tensors of a call.  Strides are in elements, rows start on 16-byte
 * boundaries.  A call has at most 2^36 - 2^12 values of x and k <= 2^30, a product rows <= 2^20 and n <= 2^29; 0 rows (and n = 0)
 * are nothing to do, and no pointer is looked at then.  `stream` is a hipStream_t as void*; calls are asynchronous on it, allocate nothing and can be captured.
 * Inputs are not written.  Results do not depend on what else runs, and equal calls give equal bits.  The return value is 0
 * or an NQX_ERR code, nqx_last_error() holds the message of the calling thread's last failure.  The reference has no
 * counterpart: its linears are 4-bit integers with 16-bit activations. */
#ifndef NQ_MX_OPS_H_
#define NQ_MX_OPS_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum nqx_dtype { NQX_F16 = 0, NQX_BF16 = 1, NQX_F32 = 2 };
enum nqx_format { NQX_FP4 = 0, NQX_FP8 = 1 };
enum nqx_status { NQX_OK = 0, NQX_ERR_ARG = 1, NQX_ERR_UNSUPPORTED = 2, NQX_ERR_WORKSPACE = 3, NQX_ERR_HIP = 4 };

const char* nqx_last_error(void);

/* codes, scales = x [rows, k], rows x_stride apart. */
int nqx_quantize(const void* x, int64_t x_stride, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t k, int dtype,
                 int format, void* stream);

/* y [rows, k] = the values that codes and scales stand for, rounded once to dtype. */
int nqx_dequantize(const uint8_t* codes, const uint8_t* scales, void* y, int64_t rows, int64_t k, int dtype, int format,
                   void* stream);

/* y [rows, n] = x . weight^T + bias for quantised x (format) and 4-bit weights: products of the elements, scaled, summed in
 * fp32; the bias [n] of type dtype (or NULL) is added in fp32 and the sum is rounded once.  (The matrix instruction of e4m3
 * with e2m1 adds eight consecutive products in fixed point, in units of 2^-13 of the largest: far below what e4m3 rounded off.
 * Of NaN codes and scales the sum is NaN.)
 * workspace: nqx_linear_workspace_bytes (0 is possible; quantised = 1), 16-byte aligned, any contents, not to be shared by calls
 * that may overlap. */
size_t nqx_linear_workspace_bytes(int64_t rows, int64_t n, int64_t k, int dtype, int format, int quantised);
int nqx_linear_quantized(const uint8_t* codes, const uint8_t* scales, const uint8_t* weight, const uint8_t* weight_scales,
                         const void* bias, void* y, int64_t rows, int64_t n, int64_t k, int dtype, int format,
                         void* workspace, size_t workspace_bytes, void* stream);

/* The same for x [rows, k] of type dtype, rows x_stride apart, quantised to `format` on the way: the codes of nqx_quantize, and
 * sums that may be added up in another order.  workspace as above, with quantised = 0. */
int nqx_linear(const void* x, int64_t x_stride, const uint8_t* weight, const uint8_t* weight_scales, const void* bias,
               void* y, int64_t rows, int64_t n, int64_t k, int dtype, int format, void* workspace, size_t workspace_bytes,
               void* stream);
/* The kernel that nqx_linear_quantized (quantised = 1) or nqx_linear (0) runs the product of these sizes on, by name. */
const char* nqx_linear_form(int64_t rows, int64_t n, int64_t k, int dtype, int format, int quantised);

/* total [rows, k] = x + delta, rounded to dtype (delta NULL: total is x, and may be NULL, else it is written too), and
 * codes, scales of total * rsqrt(mean(total^2) + eps) * weight, computed in fp32 from the rounded sum.  x, delta and total
 * are rows x_stride, delta_stride and k apart; total may be x or delta where their rows are k apart.  Squares past fp32 give a
 * mean of infinity, and zeros.  k <= 16384, rows < 2^24. */
int nqx_add_rmsnorm(const void* x, int64_t x_stride, const void* delta, int64_t delta_stride, const void* weight,
                    void* total, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t k, float eps, int dtype, int format,
                    void* stream);

/* codes, scales of SiLU(gate) * up = gate / (1 + exp(-gate)) * up, computed in fp32; where gate is far below zero as
 * gate * exp(gate) * up, so that results are kept whose exp(-gate) is past fp32.  A gate of -inf gives NaN.
 * gate and up [rows, k], rows gate_stride and up_stride apart (2 k for the halves of one tensor). */
int nqx_silu_mul(const void* gate, int64_t gate_stride, const void* up, int64_t up_stride, uint8_t* codes, uint8_t* scales,
                 int64_t rows, int64_t k, int dtype, int format, void* stream);

#ifdef __cplusplus
}
#endif
#endif
