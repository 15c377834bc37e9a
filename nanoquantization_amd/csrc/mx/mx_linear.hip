// The linear entry points of libnq_mx.so: argument checks, and which kernel runs a product.
#include "mx_linear.hpp"

using namespace nqx;

namespace {

int check_product(const char* fn, int64_t rows, int64_t n, int64_t k, int dtype, int format) {
    if (int s = check_types(fn, rows, k, dtype, format)) return s;
    if (n < 0) return refuse(NQX_ERR_ARG, "%s: n must not be negative (%lld)", fn, (long long)n);
    if (n > ((int64_t)1 << 30) || rows > ((int64_t)1 << 20))
        return refuse(NQX_ERR_UNSUPPORTED, "%s: problem too large (rows=%lld n=%lld)", fn, (long long)rows, (long long)n);
    return NQX_OK;
}

int check_operands(const char* fn, const uint8_t* weight, const uint8_t* weight_scales, const void* y) {
    if (!weight || !aligned16(weight) || !weight_scales || !y || !aligned16(y))
        return refuse(NQX_ERR_ARG, "%s: weight and y must be 16-byte aligned device pointers, and weight_scales not null", fn);
    return NQX_OK;
}

// Which kernel runs a product: 0 the one that streams the weight, else the size of a tile.
int form_of(int64_t rows, int64_t n, int64_t k, int format) {
    if (rows <= 64 || k > ((int64_t)1 << 22)) return 0;      // byte offsets in a tile are 32 bits
    return cdiv(rows, 256) * cdiv(n, 256) >= 192 ? 256 : 128;
}
int product(const Product& p, hipStream_t stream) {
    const int form = form_of(p.rows, p.n, p.k, p.format);
    return form ? tiles_product(p, form, stream) : skinny_product(p, stream);
}

// Where nqx_linear keeps the quantised x: codes, then scales.
int64_t scales_at(int64_t rows, int64_t k, int format) { return rows * code_bytes(k, format); }

}  // namespace

extern "C" int nqx_linear_quantized(const uint8_t* codes, const uint8_t* scales, const uint8_t* weight,
                                    const uint8_t* weight_scales, const void* bias, void* y, int64_t rows, int64_t n, int64_t k,
                                    int dtype, int format, void* stream) {
    const char* fn = "nqx_linear_quantized";
    if (int s = check_product(fn, rows, n, k, dtype, format)) return s;
    if (rows == 0 || n == 0) return NQX_OK;
    if (!codes || !aligned16(codes) || !scales)
        return refuse(NQX_ERR_ARG, "%s: codes must be a 16-byte aligned device pointer, and scales not null", fn);
    if (int s = check_operands(fn, weight, weight_scales, y)) return s;
    return product({codes, scales, weight, weight_scales, bias, y, rows, n, k, dtype, format}, static_cast<hipStream_t>(stream));
}

extern "C" size_t nqx_linear_workspace_bytes(int64_t rows, int64_t n, int64_t k, int dtype, int format) {
    if (check_product("nqx_linear_workspace_bytes", rows, n, k, dtype, format) || rows == 0 || n == 0) return 0;
    return (size_t)(scales_at(rows, k, format) + rows * (k / kBlock));
}

extern "C" int nqx_linear(const void* x, int64_t x_stride, const uint8_t* weight, const uint8_t* weight_scales, const void* bias,
                          void* y, int64_t rows, int64_t n, int64_t k, int dtype, int format, void* workspace,
                          size_t workspace_bytes, void* stream) {
    const char* fn = "nqx_linear";
    if (int s = check_product(fn, rows, n, k, dtype, format)) return s;
    if (rows == 0 || n == 0) return NQX_OK;
    if (int s = check_rows(fn, "x", x, x_stride, k, dtype)) return s;
    if (int s = check_operands(fn, weight, weight_scales, y)) return s;
    const size_t wanted = nqx_linear_workspace_bytes(rows, n, k, dtype, format);
    if (!workspace || !aligned16(workspace) || workspace_bytes < wanted)
        return refuse(NQX_ERR_WORKSPACE, "%s: a 16-byte aligned workspace of %zu bytes is needed, got %zu", fn, wanted, workspace ? workspace_bytes : 0);
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    uint8_t* scales = codes + scales_at(rows, k, format);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (int s = quantize(x, x_stride, codes, scales, rows, k, dtype, format, st)) return s;
    return product({codes, scales, weight, weight_scales, bias, y, rows, n, k, dtype, format}, st);
}

extern "C" const char* nqx_linear_form(int64_t rows, int64_t n, int64_t k, int dtype, int format, int) {
    if (check_product("nqx_linear_form", rows, n, k, dtype, format) || rows == 0 || n == 0) return "";
    const int form = form_of(rows, n, k, format);
    return form == 256 ? "mx_tiles_kernel 256 x 256" : form == 128 ? "mx_tiles_kernel 128 x 128" : "mx_skinny_kernel";
}
