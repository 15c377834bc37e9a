// The linear entry points of libnq_mx.so: argument checks, and which kernel runs a product.
#include "mx_linear.hpp"

using namespace nqx;

namespace {

int check_product(const char* fn, int64_t rows, int64_t n, int64_t k, int dtype, int format) {
    if (int s = check_types(fn, rows, k, dtype, format)) return s;
    if (n < 0) return refuse(NQX_ERR_ARG, "%s: n must not be negative (%lld)", fn, (long long)n);
    if (n > ((int64_t)1 << 29) || rows > ((int64_t)1 << 20))
        return refuse(NQX_ERR_UNSUPPORTED, "%s: problem too large (rows=%lld n=%lld)", fn, (long long)rows, (long long)n);
    return NQX_OK;
}

int check_operands(const char* fn, const uint8_t* weight, const uint8_t* weight_scales, const void* y) {
    if (!weight || !aligned16(weight) || !weight_scales || !y || !aligned16(y))
        return refuse(NQX_ERR_ARG, "%s: weight and y must be 16-byte aligned device pointers, and weight_scales not null", fn);
    return NQX_OK;
}

enum Form { kSkinny, kStream, kTiles128, kTiles256 };

// Which kernel runs a product.
Form form_of(int64_t rows, int64_t n, int64_t k, int format) {
    if (k > ((int64_t)1 << 22)) return kSkinny;              // byte offsets in a tile are 32 bits
    // One launch without a split while that is shorter than a split product and the launch that adds its sums.  One row by 4096 x 4096
    // 4.8 us and 8.0, by 4096 x 12288 8.5 and 9.2, by 5120 x 12288 10.0 and 9.8.  Long rows are many rounds of a few workgroups: by
    // 9728 x 1024 6.6 and 7.2, by 12288 x 1024 9.0 and 7.3, by 25600 x 256 15.4 and 8.2; and where they are a multiple of 4 KiB apart,
    // 16 of them at a time ask the same channels: by 8192 x 5120 11.0 and 9.0.  More rows, which every 16 weight rows read again:
    // e4m3 16 by 4096 x 4096 6.7 and 8.2, 8 by 2560 x 9728 7.3 and 8.9, 8 by 4096 x 8192 9.1 and 7.6, 8 by 9728 x 1024 8.6 and 7.1; e2m1
    // 16 by 2560 x 9728 7.3 and 9.0.
    const int64_t weight = n * k, Mi = (int64_t)1 << 20;
    const bool one = rows <= 4 ? k <= 10240 && weight <= 48 * Mi
                               : rows <= 16 && k <= 6144 && weight <= 24 * Mi && rows * weight <= (format == NQX_FP4 ? 512 : n >= 4096 ? 256 : 128) * Mi;
    if (one && k % 8192 != 0) return kSkinny;
    // One round of workgroups with eight waves each, while there is one: 256 tiles of 128 (1024 rows by 4096 x 4096) in 8 bits 23.3 us
    // and 28.4 by tiles; of 288 (1100 rows) 42.0 and 35.9.  Where k is not split tiles are better off in 4 bits, whose fragments they
    // read a step ahead, but for weights that take longer to come: 200 rows by 1024 x 4096 8.1 and 6.1, 1000 by 4096 x 4096 18.5 and
    // 16.0, 128 by 4096 x 12288 16.9 and 15.5, by 5120 x 12288 21.9 and 25.9.
    const bool round = rows <= 128 || cdiv(rows, 128) * cdiv(n, 128) <= 256;
    if (round && (format == NQX_FP8 || rows <= 64 || weight > 48 * Mi || stream_splits(rows, n, k, format))) return kStream;
    // Tiles of 256 need half the bytes a product, tiles of 128 waste less where the last round of workgroups is not full (two of them
    // fit a CU).  In tenths of the time of 256 tiles of 128 a round of 256 tiles of 256 takes 33 (e2m1) or 35 (e4m3), one of 512 of 128
    // 20, and a last one of up to 256 of them 13 or 11: 8192 by 4096 x 12288 in 4 bits 238 us and 288 by tiles of 128, in 8 bits 359 and
    // 410; 3151 by 1024 x 20480 75 and 61, 104 and 87; 3000 by 4096 x 4096 34.6 and 35.9, 59.3 and 54.9.
    const int64_t wide = cdiv(rows, 256) * cdiv(n, 256), small = cdiv(rows, 128) * cdiv(n, 128), last = small % 512;
    const bool four = format == NQX_FP4;
    return cdiv(wide, 256) * (four ? 33 : 35) <= small / 512 * 20 + (last == 0 ? 0 : last > 256 ? 20 : four ? 13 : 11) ? kTiles256 : kTiles128;
}
// Whether a linear quantises x in the product's own kernel, which every workgroup does for its run of k, instead of a launch in
// front of it (two microseconds or three): where that is a little.  mx_skinny_kernel with 40 KiB of LDS for it (4 rows by 9728 x
// 2560) 9.5 us and 11.7 with the launch; mx_stream_kernel with 6 KiB (6 rows by 4096 x 12288) 10.8 and 11.4, with 10 (2 rows by 5120 x
// 25600) 18.2 and 18.1, with 17 (8 rows by 2560 x 9728) 11.3 and 10.2, with 42 (8 rows by 5120 x 25600) 25.9 and 18.4.
bool raw_of(int64_t rows, int64_t n, int64_t k, int format) {
    if (rows > 16) return false;
    const Form form = form_of(rows, n, k, format);
    return form == kStream ? stream_raw_bytes(rows, n, k, format) <= 10 * 1024
                           : form == kSkinny && skinny_raw_bytes(rows, k, format) <= 48 * 1024;
}
int product(const Product& p, hipStream_t stream) {
    switch (form_of(p.rows, p.n, p.k, p.format)) {
        case kTiles256: return tiles_product(p, 256, stream);
        case kTiles128: return tiles_product(p, 128, stream);
        case kStream: return stream_product(p, stream);
        default: return skinny_product(p, stream);
    }
}

// A call's workspace: the sums of a split product, the codes of x, the scales of x.
struct Space {
    size_t sums, codes, scales;
    size_t bytes() const { return sums + codes + scales; }
};
Space space_of(int64_t rows, int64_t n, int64_t k, int format, bool quantised) {
    Space s = {0, 0, 0};
    if (rows == 0 || n == 0) return s;
    if (form_of(rows, n, k, format) == kStream) s.sums = stream_sums_bytes(rows, n, k, format);
    if (!quantised && !raw_of(rows, n, k, format)) s.codes = (size_t)(rows * code_bytes(k, format)), s.scales = (size_t)(rows * (k / kBlock));
    return s;
}
int check_space(const char* fn, size_t wanted, const void* workspace, size_t bytes) {
    if (wanted && (!workspace || !aligned16(workspace) || bytes < wanted))
        return refuse(NQX_ERR_WORKSPACE, "%s: a 16-byte aligned workspace of %zu bytes is needed, got %zu", fn, wanted, workspace ? bytes : 0);
    return NQX_OK;
}

}  // namespace

extern "C" size_t nqx_linear_workspace_bytes(int64_t rows, int64_t n, int64_t k, int dtype, int format, int quantised) {
    if (check_product("nqx_linear_workspace_bytes", rows, n, k, dtype, format)) return 0;
    return space_of(rows, n, k, format, quantised != 0).bytes();
}

extern "C" int nqx_linear_quantized(const uint8_t* codes, const uint8_t* scales, const uint8_t* weight,
                                    const uint8_t* weight_scales, const void* bias, void* y, int64_t rows, int64_t n, int64_t k,
                                    int dtype, int format, void* workspace, size_t workspace_bytes, void* stream) {
    const char* fn = "nqx_linear_quantized";
    if (int s = check_product(fn, rows, n, k, dtype, format)) return s;
    if (rows == 0 || n == 0) return NQX_OK;
    if (!codes || !aligned16(codes) || !scales)
        return refuse(NQX_ERR_ARG, "%s: codes must be a 16-byte aligned device pointer, and scales not null", fn);
    if (int s = check_operands(fn, weight, weight_scales, y)) return s;
    if (int s = check_space(fn, space_of(rows, n, k, format, true).bytes(), workspace, workspace_bytes)) return s;
    return product({codes, scales, weight, weight_scales, bias, y, rows, n, k, dtype, format, static_cast<float*>(workspace)},
                   static_cast<hipStream_t>(stream));
}

extern "C" int nqx_linear(const void* x, int64_t x_stride, const uint8_t* weight, const uint8_t* weight_scales, const void* bias,
                          void* y, int64_t rows, int64_t n, int64_t k, int dtype, int format, void* workspace,
                          size_t workspace_bytes, void* stream) {
    const char* fn = "nqx_linear";
    if (int s = check_product(fn, rows, n, k, dtype, format)) return s;
    if (rows == 0 || n == 0) return NQX_OK;
    if (int s = check_rows(fn, "x", x, x_stride, k, dtype)) return s;
    if (int s = check_operands(fn, weight, weight_scales, y)) return s;
    const Space space = space_of(rows, n, k, format, false);
    if (int s = check_space(fn, space.bytes(), workspace, workspace_bytes)) return s;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    Product p = {nullptr, nullptr, weight, weight_scales, bias, y, rows, n, k, dtype, format, static_cast<float*>(workspace)};
    if (!space.codes) {
        p.raw = x, p.raw_stride = x_stride;
        return product(p, st);
    }
    uint8_t* codes = static_cast<uint8_t*>(workspace) + space.sums;
    uint8_t* scales = codes + space.codes;
    if (int s = quantize(x, x_stride, codes, scales, rows, k, dtype, format, st)) return s;
    p.x = codes, p.xs = scales;
    return product(p, st);
}

extern "C" const char* nqx_linear_form(int64_t rows, int64_t n, int64_t k, int dtype, int format, int quantised) {
    if (check_product("nqx_linear_form", rows, n, k, dtype, format) || rows == 0 || n == 0) return "";
    switch (form_of(rows, n, k, format)) {
        case kTiles256: return "mx_tiles_kernel 256 x 256";
        case kTiles128: return "mx_tiles_kernel 128 x 128";
        case kStream: return !quantised && raw_of(rows, n, k, format) ? "mx_stream_kernel on x as it is" : "mx_stream_kernel";
        default: return !quantised && raw_of(rows, n, k, format) ? "mx_skinny_kernel on x as it is" : "mx_skinny_kernel";
    }
}
