// PyTorch-ROCm operators over the C ABI of libnq_mx.so (include/nq_mx_ops.h): torch.ops.nanoquantization_amd.mx_*.  Host
// code only.  Each checks its arguments, allocates its results from torch's allocator (the workspace of a linear too: it
// belongs to the call, so calls on several streams and captured graphs do not share it) and launches on torch's current
// stream of the tensors' device.  HIP and Meta kernels; inference only (none has a derivative), and no CPU kernel.
#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/library.h>

#include "../../../include/nq_mx_ops.h"

namespace {

using DeviceGuard = c10::hip::HIPGuardMasqueradingAsCUDA;
using Two = std::tuple<at::Tensor, at::Tensor>;
using Three = std::tuple<at::Tensor, at::Tensor, at::Tensor>;
using OptTensor = c10::optional<at::Tensor>;

constexpr int64_t kBlock = 32;

hipStream_t stream_of(const at::Tensor& t) {
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}
void check_status(int status, const char* entry) {
    TORCH_CHECK(status == NQX_OK, "libnq_mx: ", entry, " failed (status ", status, "): ", nqx_last_error());
}
int dtype_id(at::ScalarType t) {
    TORCH_CHECK(t == at::kHalf || t == at::kBFloat16 || t == at::kFloat, "float16, bfloat16 or float32 expected, got ", t);
    return t == at::kHalf ? NQX_F16 : t == at::kBFloat16 ? NQX_BF16 : NQX_F32;
}
int format_id(c10::string_view f) {
    TORCH_CHECK(f == "mxfp4" || f == "mxfp8", "the format must be 'mxfp4' or 'mxfp8', got '", f, "'");
    return f == "mxfp4" ? NQX_FP4 : NQX_FP8;
}
void check_device(const at::Tensor& ref, std::initializer_list<const at::Tensor*> others) {
    for (const at::Tensor* t : others)
        TORCH_CHECK(t->device() == ref.device(), "tensors on different devices: ", t->device(), " vs ", ref.device());
}
bool off16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) != 0; }
at::Tensor dense16(const at::Tensor& t) {
    const at::Tensor d = t.contiguous();
    return off16(d) ? d.clone() : d;
}

// A tensor as rows of its last dimension, read in place where the rows are dense and start on 16-byte boundaries.
struct Rows {
    at::Tensor t;
    int64_t rows, k, stride;
};
int64_t last_size(const at::Tensor& x, const char* what) {
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0 && x.size(-1) % kBlock == 0, what, " must have a last dimension that is a positive multiple of ",
                kBlock, ", got ", x.sizes());
    return x.size(-1);
}
Rows rows_of(const at::Tensor& x) {
    const int64_t k = x.size(-1);
    at::Tensor t = x.dim() == 2 ? x : x.reshape({x.numel() / k, k});
    const int64_t rows = t.size(0), bytes = t.element_size();
    if (rows && (t.stride(1) != 1 || off16(t) || (rows > 1 && t.stride(0) * bytes % 16 != 0))) t = dense16(t);
    return {t, rows, k, rows > 1 ? t.stride(0) : k};
}

at::DimVector with_last(const at::Tensor& x, int64_t last) {
    at::DimVector s(x.sizes());
    s.back() = last;
    return s;
}
// An empty tensor beside x: on a HIP device by the allocator's own function, without the dispatcher's round.
at::Tensor empty_beside(const at::Tensor& x, at::IntArrayRef sizes, at::ScalarType dtype) {
    if (x.is_cuda()) return at::detail::empty_cuda(sizes, dtype, x.device(), c10::nullopt);
    return at::empty(sizes, x.options().dtype(dtype));
}
Two packed_like(const at::Tensor& x, int format) {
    const int64_t k = x.size(-1);
    return {empty_beside(x, with_last(x, format == NQX_FP4 ? k / 2 : k), at::kByte), empty_beside(x, with_last(x, k / kBlock), at::kByte)};
}

// The values a row of codes and scales stands for, and its format, which follows from the two sizes.
struct Packed {
    int64_t k;
    int format;
};
Packed check_packed(const at::Tensor& codes, const at::Tensor& scales, const char* what) {
    TORCH_CHECK(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte, what, ": codes and scales must be uint8");
    TORCH_CHECK(codes.dim() >= 1 && codes.dim() == scales.dim() && codes.sizes().slice(0, codes.dim() - 1) == scales.sizes().slice(0, scales.dim() - 1),
                what, ": codes and scales must have the same leading dimensions, got ", codes.sizes(), " and ", scales.sizes());
    const int64_t blocks = scales.size(-1), c = codes.size(-1);
    TORCH_CHECK(blocks > 0 && (c == blocks * 16 || c == blocks * 32), what,
                ": a scale goes with 16 bytes of codes (mxfp4) or 32 (mxfp8), got ", codes.sizes(), " and ", scales.sizes());
    return {blocks * kBlock, c == blocks * 16 ? NQX_FP4 : NQX_FP8};
}
int64_t check_weight(const at::Tensor& weight, const at::Tensor& weight_scales, int64_t k) {
    const Packed w = check_packed(weight, weight_scales, "weight");
    TORCH_CHECK(weight.dim() == 2 && w.format == NQX_FP4, "weight must be [n, k / 2] of mxfp4, got ", weight.sizes());
    TORCH_CHECK(w.k == k, "weight has ", w.k, " input features, and x ", k);
    return weight.size(0);
}
// Whether there is a bias, which fits then.
bool check_bias(const OptTensor& bias, const at::Tensor& x, int64_t n) {
    if (!bias.has_value() || !bias->defined()) return false;
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == n, "bias must have ", n, " elements, got ", bias->sizes());
    check_device(x, {&*bias});
    return true;
}
at::Tensor dense_bias(const OptTensor& bias, const at::Tensor& x, int64_t n, at::ScalarType dtype) {
    return check_bias(bias, x, n) ? bias->to(dtype).contiguous() : at::Tensor();
}

Two mx_quantize(const at::Tensor& x, c10::string_view format) {
    const int f = format_id(format), d = dtype_id(x.scalar_type());
    last_size(x, "x");
    const DeviceGuard guard(x.device());
    Two out = packed_like(x, f);
    if (x.numel() == 0) return out;
    const Rows r = rows_of(x);
    check_status(nqx_quantize(r.t.data_ptr(), r.stride, std::get<0>(out).data_ptr<uint8_t>(), std::get<1>(out).data_ptr<uint8_t>(), r.rows,
                              r.k, d, f, stream_of(x)),
                 "nqx_quantize");
    return out;
}
Two mx_quantize_meta(const at::Tensor& x, c10::string_view format) {
    dtype_id(x.scalar_type());
    last_size(x, "x");
    return packed_like(x, format_id(format));
}

at::Tensor mx_dequantize(const at::Tensor& codes, const at::Tensor& scales, at::ScalarType dtype) {
    const Packed p = check_packed(codes, scales, "mx_dequantize");
    const int d = dtype_id(dtype);
    check_device(codes, {&scales});
    const DeviceGuard guard(codes.device());
    at::Tensor y = empty_beside(codes, with_last(codes, p.k), dtype);
    if (y.numel() == 0) return y;
    const at::Tensor c = dense16(codes), s = scales.contiguous();
    check_status(nqx_dequantize(c.data_ptr<uint8_t>(), s.data_ptr<uint8_t>(), y.data_ptr(), y.numel() / p.k, p.k, d, p.format, stream_of(codes)),
                 "nqx_dequantize");
    return y;
}
at::Tensor mx_dequantize_meta(const at::Tensor& codes, const at::Tensor& scales, at::ScalarType dtype) {
    dtype_id(dtype);
    const Packed p = check_packed(codes, scales, "mx_dequantize");
    check_device(codes, {&scales});
    return empty_beside(codes, with_last(codes, p.k), dtype);
}

at::Tensor mx_linear(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& weight_scales, const OptTensor& bias,
                     c10::string_view activations) {
    const int f = format_id(activations), d = dtype_id(x.scalar_type());
    const int64_t k = last_size(x, "x"), n = check_weight(weight, weight_scales, k);
    check_device(x, {&weight, &weight_scales});
    const DeviceGuard guard(x.device());
    at::Tensor y = empty_beside(x, with_last(x, n), x.scalar_type());
    const at::Tensor b = dense_bias(bias, x, n, x.scalar_type());
    if (y.numel() == 0) return y;
    const Rows r = rows_of(x);
    const at::Tensor w = dense16(weight), ws = weight_scales.contiguous();
    const size_t bytes = nqx_linear_workspace_bytes(r.rows, n, k, d, f, 0);
    const at::Tensor space = bytes ? empty_beside(w, {(int64_t)bytes}, at::kByte) : at::Tensor();
    check_status(nqx_linear(r.t.data_ptr(), r.stride, w.data_ptr<uint8_t>(), ws.data_ptr<uint8_t>(), b.defined() ? b.data_ptr() : nullptr,
                            y.data_ptr(), r.rows, n, k, d, f, bytes ? space.data_ptr() : nullptr, bytes, stream_of(x)),
                 "nqx_linear");
    return y;
}
at::Tensor mx_linear_meta(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& weight_scales, const OptTensor& bias,
                          c10::string_view activations) {
    format_id(activations);
    dtype_id(x.scalar_type());
    const int64_t n = check_weight(weight, weight_scales, last_size(x, "x"));
    check_device(x, {&weight, &weight_scales});
    check_bias(bias, x, n);
    return empty_beside(x, with_last(x, n), x.scalar_type());
}

at::Tensor mx_linear_quantized(const at::Tensor& codes, const at::Tensor& scales, const at::Tensor& weight, const at::Tensor& weight_scales,
                               const OptTensor& bias, at::ScalarType dtype) {
    const Packed p = check_packed(codes, scales, "x");
    const int d = dtype_id(dtype);
    const int64_t n = check_weight(weight, weight_scales, p.k);
    check_device(codes, {&scales, &weight, &weight_scales});
    const DeviceGuard guard(codes.device());
    at::Tensor y = empty_beside(codes, with_last(codes, n), dtype);
    const at::Tensor b = dense_bias(bias, codes, n, dtype);
    if (y.numel() == 0) return y;
    const at::Tensor c = dense16(codes), s = scales.contiguous(), w = dense16(weight), ws = weight_scales.contiguous();
    const int64_t rows = y.numel() / n;
    const size_t bytes = nqx_linear_workspace_bytes(rows, n, p.k, d, p.format, 1);
    const at::Tensor space = bytes ? empty_beside(w, {(int64_t)bytes}, at::kByte) : at::Tensor();
    check_status(nqx_linear_quantized(c.data_ptr<uint8_t>(), s.data_ptr<uint8_t>(), w.data_ptr<uint8_t>(), ws.data_ptr<uint8_t>(),
                                      b.defined() ? b.data_ptr() : nullptr, y.data_ptr(), rows, n, p.k, d, p.format,
                                      bytes ? space.data_ptr() : nullptr, bytes, stream_of(codes)),
                 "nqx_linear_quantized");
    return y;
}
at::Tensor mx_linear_quantized_meta(const at::Tensor& codes, const at::Tensor& scales, const at::Tensor& weight,
                                    const at::Tensor& weight_scales, const OptTensor& bias, at::ScalarType dtype) {
    dtype_id(dtype);
    const int64_t n = check_weight(weight, weight_scales, check_packed(codes, scales, "x").k);
    check_device(codes, {&scales, &weight, &weight_scales});
    check_bias(bias, codes, n);
    return empty_beside(codes, with_last(codes, n), dtype);
}

void check_norm(const at::Tensor& x, const at::Tensor& weight) {
    const int64_t k = last_size(x, "x");
    TORCH_CHECK(k <= 16384, "rows of at most 16384 values, got ", k);
    TORCH_CHECK(weight.dim() == 1 && weight.size(0) == k && weight.scalar_type() == x.scalar_type(), "weight must be [", k, "] of x's dtype");
}
void check_alike(const at::Tensor& x, const at::Tensor& other, const char* what) {
    TORCH_CHECK(other.sizes() == x.sizes() && other.scalar_type() == x.scalar_type(), what, " must be of one size and dtype, got ", x.sizes(),
                " ", x.scalar_type(), " and ", other.sizes(), " ", other.scalar_type());
}
// delta undefined: the norm alone; total, where defined, is a dense tensor like x.
Two norm(const at::Tensor& x, const at::Tensor& delta, const at::Tensor& weight, double eps, int f, const at::Tensor& total) {
    Two out = packed_like(x, f);
    if (x.numel() == 0) return out;
    const Rows r = rows_of(x);
    const Rows e = delta.defined() ? rows_of(delta) : Rows{};
    const at::Tensor w = dense16(weight);
    check_status(nqx_add_rmsnorm(r.t.data_ptr(), r.stride, delta.defined() ? e.t.data_ptr() : nullptr, e.stride, w.data_ptr(),
                                 total.defined() ? total.data_ptr() : nullptr, std::get<0>(out).data_ptr<uint8_t>(),
                                 std::get<1>(out).data_ptr<uint8_t>(), r.rows, r.k, (float)eps, dtype_id(x.scalar_type()), f, stream_of(x)),
                 "nqx_add_rmsnorm");
    return out;
}
Three mx_add_rmsnorm(const at::Tensor& x, const at::Tensor& delta, const at::Tensor& weight, double eps, c10::string_view format) {
    const int f = format_id(format);
    dtype_id(x.scalar_type());
    check_norm(x, weight);
    check_alike(x, delta, "x and delta");
    check_device(x, {&delta, &weight});
    const DeviceGuard guard(x.device());
    const at::Tensor total = empty_beside(x, x.sizes(), x.scalar_type());
    Two out = norm(x, delta, weight, eps, f, total);
    return {std::get<0>(out), std::get<1>(out), total};
}
Three mx_add_rmsnorm_meta(const at::Tensor& x, const at::Tensor& delta, const at::Tensor& weight, double, c10::string_view format) {
    dtype_id(x.scalar_type());
    check_norm(x, weight);
    check_alike(x, delta, "x and delta");
    check_device(x, {&delta, &weight});
    Two out = packed_like(x, format_id(format));
    return {std::get<0>(out), std::get<1>(out), empty_beside(x, x.sizes(), x.scalar_type())};
}
Two mx_rmsnorm(const at::Tensor& x, const at::Tensor& weight, double eps, c10::string_view format) {
    const int f = format_id(format);
    dtype_id(x.scalar_type());
    check_norm(x, weight);
    check_device(x, {&weight});
    const DeviceGuard guard(x.device());
    return norm(x, {}, weight, eps, f, {});
}
Two mx_rmsnorm_meta(const at::Tensor& x, const at::Tensor& weight, double, c10::string_view format) {
    dtype_id(x.scalar_type());
    check_norm(x, weight);
    check_device(x, {&weight});
    return packed_like(x, format_id(format));
}

Two mx_silu_mul(const at::Tensor& gate, const at::Tensor& up, c10::string_view format) {
    const int f = format_id(format), d = dtype_id(gate.scalar_type());
    last_size(gate, "gate");
    check_alike(gate, up, "gate and up");
    check_device(gate, {&up});
    const DeviceGuard guard(gate.device());
    Two out = packed_like(gate, f);
    if (gate.numel() == 0) return out;
    const Rows g = rows_of(gate), u = rows_of(up);
    check_status(nqx_silu_mul(g.t.data_ptr(), g.stride, u.t.data_ptr(), u.stride, std::get<0>(out).data_ptr<uint8_t>(),
                              std::get<1>(out).data_ptr<uint8_t>(), g.rows, g.k, d, f, stream_of(gate)),
                 "nqx_silu_mul");
    return out;
}
Two mx_silu_mul_meta(const at::Tensor& gate, const at::Tensor& up, c10::string_view format) {
    dtype_id(gate.scalar_type());
    last_size(gate, "gate");
    check_alike(gate, up, "gate and up");
    check_device(gate, {&up});
    return packed_like(gate, format_id(format));
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(nanoquantization_amd, m) {
    m.def("mx_quantize(Tensor x, str format) -> (Tensor, Tensor)");
    m.def("mx_dequantize(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor");
    m.def("mx_linear(Tensor x, Tensor weight, Tensor weight_scales, Tensor? bias, str activations) -> Tensor");
    m.def("mx_linear_quantized(Tensor codes, Tensor scales, Tensor weight, Tensor weight_scales, Tensor? bias, ScalarType dtype) -> Tensor");
    m.def("mx_add_rmsnorm(Tensor x, Tensor delta, Tensor weight, float eps, str format) -> (Tensor, Tensor, Tensor)");
    m.def("mx_rmsnorm(Tensor x, Tensor weight, float eps, str format) -> (Tensor, Tensor)");
    m.def("mx_silu_mul(Tensor gate, Tensor up, str format) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(nanoquantization_amd, CUDA, m) {   // the dispatch key of HIP tensors in PyTorch-ROCm
    m.impl("mx_quantize", &mx_quantize);
    m.impl("mx_dequantize", &mx_dequantize);
    m.impl("mx_linear", &mx_linear);
    m.impl("mx_linear_quantized", &mx_linear_quantized);
    m.impl("mx_add_rmsnorm", &mx_add_rmsnorm);
    m.impl("mx_rmsnorm", &mx_rmsnorm);
    m.impl("mx_silu_mul", &mx_silu_mul);
}

TORCH_LIBRARY_IMPL(nanoquantization_amd, Meta, m) {
    m.impl("mx_quantize", &mx_quantize_meta);
    m.impl("mx_dequantize", &mx_dequantize_meta);
    m.impl("mx_linear", &mx_linear_meta);
    m.impl("mx_linear_quantized", &mx_linear_quantized_meta);
    m.impl("mx_add_rmsnorm", &mx_add_rmsnorm_meta);
    m.impl("mx_rmsnorm", &mx_rmsnorm_meta);
    m.impl("mx_silu_mul", &mx_silu_mul_meta);
}
