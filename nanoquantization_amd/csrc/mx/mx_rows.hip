// Row kernels of the microscaled formats: quantise, dequantise, residual addition + RMSNorm, SiLU(gate) * up.  All are
// bound by memory: a lane takes eight consecutive values in one or two 16-byte loads, several eights at once, the four lanes of
// a block agree on the largest magnitude by two DPP moves, and codes leave in 4- or 8-byte stores, whole lines a wave.  In bf16, on
// tensors that are in no cache, 25600 x 5120: quantise to e2m1 59 us, to e4m3 70 (5.6 and 5.7 TB/s), dequantise 59 and 68 (5.6 and
// 5.8); 8192 x 5120: sum, norm and e4m3 54 us (5.4 TB/s); 8192 x 12288: SiLU to e2m1 84 us (5.5 TB/s).  A large copy reaches 5.1.
#include "mx_common.hpp"

namespace nqx {
namespace {

constexpr int kThreads = 256;

// A workgroup takes kMany * 256 consecutive eights of the tensor, a lane kMany of them, all loaded before the first is used.
constexpr int kMany = 4;

// Where eight `at` of rows `stride` values apart begins.  Dense rows need no division, which would cost a launch of a few rows a
// microsecond; others, of fewer than 2^31 eights, one by a product: with 2^(bits - 1) < per_row <= 2^bits and magic =
// 2^(31 + bits) / per_row rounded up, at * magic / 2^(31 + bits) is past at / per_row by less than 1 / per_row.
struct Rows {
    uint32_t per_row, magic, bits;           // magic 0: 2^31 eights or more
};
Rows rows_of(int64_t count, int64_t k) {
    Rows r = {(uint32_t)(k / kLane), 0, 0};
    while ((1u << r.bits) < r.per_row) ++r.bits;
    if (count < ((int64_t)1 << 31)) r.magic = (uint32_t)((((uint64_t)1 << (31 + r.bits)) + r.per_row - 1) / r.per_row);
    return r;
}
__device__ __forceinline__ int64_t place(int64_t at, int64_t stride, Rows r) {
    if (stride == (int64_t)r.per_row * 8) return at * 8;
    if (r.magic) {
        const uint32_t row = __umulhi((uint32_t)at, r.magic) >> (r.bits - 1);
        return row * stride + (int64_t)((uint32_t)at - row * r.per_row) * 8;
    }
    const int64_t row = at / r.per_row;
    return row * stride + (at - row * r.per_row) * 8;
}

template <typename T, int FORMAT>
__global__ __launch_bounds__(kThreads) void mx_quantize_kernel(const typename T::elem* __restrict__ x, int64_t stride,
                                                               uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                               int64_t count, Rows in) {
    const int64_t first = (int64_t)blockIdx.x * (kMany * kThreads) + threadIdx.x;
    Eight<T, FORMAT> e[kMany];
#pragma unroll
    for (int u = 0; u < kMany; ++u) {
        const int64_t at = first + u * kThreads;
        if (at < count) e[u].load(x + place(at, stride, in));
    }
#pragma unroll
    for (int u = 0; u < kMany; ++u) {
        const int64_t at = first + u * kThreads;
        if (at >= count) break;              // whole blocks: count is a multiple of four
        uint32_t byte;
        const u32x2 code = e[u].encode(byte);
        put8<FORMAT>(code, byte, codes, scales, at);
    }
}

template <typename T, int FORMAT>
__global__ __launch_bounds__(kThreads) void mx_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                                 const uint8_t* __restrict__ scales,
                                                                 typename T::elem* __restrict__ y, int64_t count) {
    const int64_t first = (int64_t)blockIdx.x * (kMany * kThreads) + threadIdx.x;
    u32x2 w[kMany];
    uint32_t byte[kMany];
#pragma unroll
    for (int u = 0; u < kMany; ++u) {
        const int64_t at = first + u * kThreads;
        w[u] = u32x2{0u, 0u}, byte[u] = 0;
        if (at >= count) continue;
        if constexpr (FORMAT == NQX_FP4) w[u].x = reinterpret_cast<const uint32_t*>(codes)[at];
        else w[u] = reinterpret_cast<const u32x2*>(codes)[at];
        byte[u] = scales[at >> 2];
    }
#pragma unroll
    for (int u = 0; u < kMany; ++u) {
        const int64_t at = first + u * kThreads;
        if (at >= count) break;
        const float scale = power(byte[u]);
        float v[8];
        // element times power of two is exact in fp32
        if constexpr (FORMAT == NQX_FP4) {
            const auto two = [&](auto sel) {
                const auto p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u].x, 1.0f, decltype(sel)::value);
                v[2 * decltype(sel)::value] = p[0] * scale, v[2 * decltype(sel)::value + 1] = p[1] * scale;
            };
            two(Const<0>()), two(Const<1>()), two(Const<2>()), two(Const<3>());
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w[u][i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w[u][i], true);
                v[4 * i] = a[0] * scale, v[4 * i + 1] = a[1] * scale, v[4 * i + 2] = b[0] * scale, v[4 * i + 3] = b[1] * scale;
            }
        }
        store8<T>(y + at * 8, v);
    }
}

// One row a workgroup, kept in registers between the statistics and the result: CHUNKS eights a lane.
template <typename T, int FORMAT, int CHUNKS>
__global__ __launch_bounds__(kThreads) void mx_add_rmsnorm_kernel(const typename T::elem* x, int64_t x_stride,
                                                                  const typename T::elem* delta, int64_t delta_stride,
                                                                  const typename T::elem* __restrict__ weight,
                                                                  typename T::elem* total, uint8_t* __restrict__ codes,
                                                                  uint8_t* __restrict__ scales, uint32_t per_row, float eps) {
    __shared__ float s_sum[kThreads / 64];
    const int64_t row = blockIdx.x;
    Eight<T, FORMAT> in[CHUNKS], add[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const uint32_t column = c * kThreads + threadIdx.x;
        in[c].clear(), add[c].clear();
        if (column < per_row) {
            in[c].load(x + row * x_stride + (int64_t)column * 8);
            if (delta) add[c].load(delta + row * delta_stride + (int64_t)column * 8);
        }
    }
    float v[CHUNKS][8], ss = 0.f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const uint32_t column = c * kThreads + threadIdx.x;
        in[c].floats(v[c]);
        if (delta) {
            float d[8];
            add[c].floats(d);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[c][e] = T::to_f32(T::from_f32(v[c][e] + d[e]));
        }
        if (total && column < per_row) store8<T>(total + (row * per_row + column) * 8, v[c]);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(v[c][e], v[c][e], ss);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) ss += __shfl_xor(ss, o);
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) ss += s_sum[w];
    const float r = 1.0f / sqrtf(ss / (float)(per_row * 8) + eps);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const uint32_t column = c * kThreads + threadIdx.x;
        if (column < per_row) {         // whole blocks: a row has a multiple of four eights
            float w[8];
            load8<T>(weight + (int64_t)column * 8, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[c][e] = v[c][e] * r * w[e];
            quantize8<FORMAT>(v[c], codes, scales, row * per_row + column);
        }
    }
}

// gate / (1 + exp(-gate)) * up.  exp(-g) is 2^t 2^r, t = -g log2(e) rounded and r what that and the constant lost: without r the
// relative error grows with |g|.  (2^r as a factor of its own near 1: where 2^t is infinite a sum could be inf - inf.)  The
// reciprocal is off by a step of fp32 at most, a division would be by half of one and takes ten times as long (8192 x 12288 bf16
// to e2m1 is 84 us, and 97 with expf and a division; to e4m3 91 and 103).  Above 100 the exponential does not change 1.  For gates
// below kFar the result is silu_mul_far's: the hardware reciprocal has no subnormal results, so from -87.3 on it would be 0, which a
// large `up` would make of values that are not small.
constexpr float kHigh = 1.44269502f, kLow = 1.92596303e-8f;       // log2(e) in two parts
constexpr float kFar = -80.f;
__device__ __forceinline__ float silu_mul(float gate, float up) {
    constexpr float kLn2 = 0.693147182f;
    const float g = -__builtin_amdgcn_fmed3f(gate, -100.f, 100.f), t = g * kHigh;
    const float r = __builtin_fmaf(g, kLow, __builtin_fmaf(g, kHigh, -t));
    const float e = __builtin_amdgcn_exp2f(t) * __builtin_fmaf(r, kLn2, 1.0f);
    return gate * __builtin_amdgcn_rcpf(1.0f + e) * up;
}
// The same for gates below kFar, where 1 + exp(-gate) is exp(-gate) in fp32: gate * exp(gate) * up, its powers of two last, so that
// nothing under- or overflows that the result does not.  exp(gate) is 2^n 2^f, n = gate log2(e) rounded to a whole number.  (Gates below
// -1000 are 0 times any `up`; -inf stays, a NaN as inf / inf is.)
__device__ __forceinline__ float silu_mul_far(float gate, float up) {
    const float g = fmaxf(gate, -1000.f), n = __builtin_rintf(g * kHigh);
    const float f = __builtin_fmaf(g, kLow, __builtin_fmaf(g, kHigh, -n));
    const float m = g * __builtin_amdgcn_exp2f(f) * __builtin_amdgcn_frexp_mantf(up);
    return gate == -__builtin_inff() ? __builtin_nanf("") : __builtin_ldexpf(m, (int)n + __builtin_amdgcn_frexp_expf(up));
}

template <typename T, int FORMAT>
__global__ __launch_bounds__(kThreads) void mx_silu_mul_kernel(const typename T::elem* __restrict__ gate, int64_t gate_stride,
                                                               const typename T::elem* __restrict__ up, int64_t up_stride,
                                                               uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                               int64_t count, Rows in) {
    constexpr int kTwo = 2;                  // eights of a lane: they are two loads each
    const int64_t first = (int64_t)blockIdx.x * (kTwo * kThreads) + threadIdx.x;
    Eight<T, FORMAT> g[kTwo], u[kTwo];
#pragma unroll
    for (int i = 0; i < kTwo; ++i) {
        const int64_t at = first + i * kThreads;
        if (at < count) g[i].load(gate + place(at, gate_stride, in)), u[i].load(up + place(at, up_stride, in));
    }
#pragma unroll
    for (int i = 0; i < kTwo; ++i) {
        const int64_t at = first + i * kThreads;
        if (at >= count) break;
        float a[8], b[8];
        g[i].floats(a), u[i].floats(b);
        float v[8], least = a[0];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = silu_mul(a[e], b[e]), least = fminf(least, a[e]);
        if (least < kFar) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (a[e] < kFar) v[e] = silu_mul_far(a[e], b[e]);
        }
        quantize8<FORMAT>(v, codes, scales, at);
    }
}

unsigned groups(int64_t eights, int of_a_lane) { return (unsigned)cdiv(eights, of_a_lane * kThreads); }

}  // namespace

int quantize(const void* x, int64_t x_stride, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t k, int dtype, int format,
             hipStream_t stream) {
    hipError_t e = hipSuccess;
    by_type(dtype, format, [&](auto t, auto f) {
        using T = decltype(t);
        const int64_t count = rows * (k / kLane);
        e = start(&mx_quantize_kernel<T, decltype(f)::value>, dim3(groups(count, kMany)), kThreads, 0, stream,
            static_cast<const typename T::elem*>(x), x_stride, codes, scales, count, rows_of(count, k));
    });
    return hip_status("nqx_quantize", e);
}

}  // namespace nqx

using namespace nqx;

static int check_out(const char* fn, const uint8_t* codes, const uint8_t* scales) {
    if (!codes || !aligned16(codes) || !scales) return refuse(NQX_ERR_ARG, "%s: codes must be a 16-byte aligned device pointer, and scales not null", fn);
    return NQX_OK;
}

extern "C" int nqx_quantize(const void* x, int64_t x_stride, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t k, int dtype,
                            int format, void* stream) {
    if (int s = check_types("nqx_quantize", rows, k, dtype, format)) return s;
    if (rows == 0) return NQX_OK;
    if (int s = check_rows("nqx_quantize", "x", x, x_stride, k, dtype)) return s;
    if (int s = check_out("nqx_quantize", codes, scales)) return s;
    return quantize(x, x_stride, codes, scales, rows, k, dtype, format, static_cast<hipStream_t>(stream));
}

extern "C" int nqx_dequantize(const uint8_t* codes, const uint8_t* scales, void* y, int64_t rows, int64_t k, int dtype, int format,
                              void* stream) {
    if (int s = check_types("nqx_dequantize", rows, k, dtype, format)) return s;
    if (rows == 0) return NQX_OK;
    if (int s = check_rows("nqx_dequantize", "y", y, k, k, dtype)) return s;
    if (int s = check_out("nqx_dequantize", codes, scales)) return s;
    hipError_t e = hipSuccess;
    by_type(dtype, format, [&](auto t, auto f) {
        using T = decltype(t);
        const int64_t count = rows * (k / kLane);
        e = start(&mx_dequantize_kernel<T, decltype(f)::value>, dim3(groups(count, kMany)), kThreads, 0, static_cast<hipStream_t>(stream),
            codes, scales, static_cast<typename T::elem*>(y), count);
    });
    return hip_status("nqx_dequantize", e);
}

extern "C" int nqx_add_rmsnorm(const void* x, int64_t x_stride, const void* delta, int64_t delta_stride, const void* weight,
                               void* total, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t k, float eps, int dtype,
                               int format, void* stream) {
    const char* fn = "nqx_add_rmsnorm";
    if (int s = check_types(fn, rows, k, dtype, format)) return s;
    if (k > 16384) return refuse(NQX_ERR_UNSUPPORTED, "%s: k must be at most 16384, got %lld", fn, (long long)k);
    if (rows >= ((int64_t)1 << 24)) return refuse(NQX_ERR_UNSUPPORTED, "%s: fewer than 2^24 rows at a time, got %lld", fn, (long long)rows);
    if (rows == 0) return NQX_OK;
    if (int s = check_rows(fn, "x", x, x_stride, k, dtype)) return s;
    if (delta) {
        if (int s = check_rows(fn, "delta", delta, delta_stride, k, dtype)) return s;
        if (!total) return refuse(NQX_ERR_ARG, "%s: with a delta, total must not be null", fn);
    }
    if (int s = check_rows(fn, "weight", weight, 0, k, dtype)) return s;
    if (total) {
        if (int s = check_rows(fn, "total", total, k, k, dtype)) return s;
        if ((total == x && x_stride != k) || (total == delta && delta_stride != k))
            return refuse(NQX_ERR_ARG, "%s: total can be x or delta only where their rows are k apart", fn);
    }
    if (int s = check_out(fn, codes, scales)) return s;
    hipError_t e = hipSuccess;
    by_type(dtype, format, [&](auto t, auto f) {
        using T = decltype(t);
        using E = typename T::elem;
        const auto with = [&](auto chunks) {
            e = start(&mx_add_rmsnorm_kernel<T, decltype(f)::value, decltype(chunks)::value>, dim3((unsigned)rows), kThreads, 0, static_cast<hipStream_t>(stream),
                    static_cast<const E*>(x), x_stride, static_cast<const E*>(delta), delta_stride, static_cast<const E*>(weight),
                    static_cast<E*>(total), codes, scales, (uint32_t)(k / kLane), eps);
        };
        const int64_t chunks = cdiv(k / kLane, kThreads);
        if (chunks <= 1) with(Const<1>());
        else if (chunks <= 2) with(Const<2>());
        else if (chunks <= 3) with(Const<3>());
        else if (chunks <= 4) with(Const<4>());
        else with(Const<8>());
    });
    return hip_status(fn, e);
}

extern "C" int nqx_silu_mul(const void* gate, int64_t gate_stride, const void* up, int64_t up_stride, uint8_t* codes,
                            uint8_t* scales, int64_t rows, int64_t k, int dtype, int format, void* stream) {
    const char* fn = "nqx_silu_mul";
    if (int s = check_types(fn, rows, k, dtype, format)) return s;
    if (rows == 0) return NQX_OK;
    if (int s = check_rows(fn, "gate", gate, gate_stride, k, dtype)) return s;
    if (int s = check_rows(fn, "up", up, up_stride, k, dtype)) return s;
    if (int s = check_out(fn, codes, scales)) return s;
    hipError_t e = hipSuccess;
    by_type(dtype, format, [&](auto t, auto f) {
        using T = decltype(t);
        using E = typename T::elem;
        const int64_t count = rows * (k / kLane);
        e = start(&mx_silu_mul_kernel<T, decltype(f)::value>, dim3(groups(count, 2)), kThreads, 0, static_cast<hipStream_t>(stream),
            static_cast<const E*>(gate), gate_stride, static_cast<const E*>(up), up_stride, codes, scales, count,
            rows_of(count, k));
    });
    return hip_status(fn, e);
}
