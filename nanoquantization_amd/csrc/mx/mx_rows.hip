// Row kernels of the microscaled formats: quantise, dequantise, residual addition + RMSNorm, SiLU(gate) * up.  All are
// bound by memory: a lane takes eight consecutive values in one or two 16-byte loads, the four lanes of a block agree on
// the largest magnitude by two DPP moves, and codes leave in 4- or 8-byte stores, whole lines a wave.
#include "mx_common.hpp"

namespace nqx {
namespace {

constexpr int kThreads = 256;

// A grid-stride loop over the tensor's eights: fn(row, column in eights, number).
template <typename F>
__device__ __forceinline__ void each_eight(int64_t count, uint32_t per_row, F&& fn) {
    for (int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x; at < count; at += (int64_t)gridDim.x * kThreads) {
        const int64_t row = at / per_row;
        fn(row, (uint32_t)(at - row * per_row), at);
    }
}

template <typename T, int FORMAT>
__global__ __launch_bounds__(kThreads) void mx_quantize_kernel(const typename T::elem* __restrict__ x, int64_t stride,
                                                               uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                               int64_t count, uint32_t per_row) {
    each_eight(count, per_row, [&](int64_t row, uint32_t column, int64_t at) {
        float v[8];
        load8<T>(x + row * stride + (int64_t)column * 8, v);
        quantize8<FORMAT>(v, codes, scales, at);
    });
}

template <typename T, int FORMAT>
__global__ __launch_bounds__(kThreads) void mx_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                                 const uint8_t* __restrict__ scales,
                                                                 typename T::elem* __restrict__ y, int64_t count) {
    for (int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x; at < count; at += (int64_t)gridDim.x * kThreads) {
        const float scale = power(scales[at >> 2]);
        float v[8];
        // element times power of two is exact in fp32
        if constexpr (FORMAT == NQX_FP4) {
            const uint32_t w = reinterpret_cast<const uint32_t*>(codes)[at];
            const auto two = [&](auto sel) {
                const auto p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, decltype(sel)::value);
                v[2 * decltype(sel)::value] = p[0] * scale, v[2 * decltype(sel)::value + 1] = p[1] * scale;
            };
            two(Const<0>()), two(Const<1>()), two(Const<2>()), two(Const<3>());
        } else {
            const u32x2 w = reinterpret_cast<const u32x2*>(codes)[at];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
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
    float v[CHUNKS][8], ss = 0.f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const uint32_t column = c * kThreads + threadIdx.x;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
        if (column < per_row) load8<T>(x + row * x_stride + (int64_t)column * 8, v[c]);
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const uint32_t column = c * kThreads + threadIdx.x;
        if (column < per_row) {
            if (delta) {
                float d[8];
                load8<T>(delta + row * delta_stride + (int64_t)column * 8, d);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[c][e] = T::to_f32(T::from_f32(v[c][e] + d[e]));
            }
            if (total) store8<T>(total + (row * per_row + column) * 8, v[c]);
        }
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

template <typename T, int FORMAT>
__global__ __launch_bounds__(kThreads) void mx_silu_mul_kernel(const typename T::elem* __restrict__ gate, int64_t gate_stride,
                                                               const typename T::elem* __restrict__ up, int64_t up_stride,
                                                               uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                               int64_t count, uint32_t per_row) {
    each_eight(count, per_row, [&](int64_t row, uint32_t column, int64_t at) {
        float g[8], u[8];
        load8<T>(gate + row * gate_stride + (int64_t)column * 8, g);
        load8<T>(up + row * up_stride + (int64_t)column * 8, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = g[e] / (1.0f + expf(-g[e])) * u[e];
        quantize8<FORMAT>(g, codes, scales, at);
    });
}

// Enough workgroups to fill the chip several times over, each with a few rounds of the loop at the largest sizes.
int grid_for(int64_t eights) {
    const int64_t g = cdiv(eights, kThreads);
    return (int)(g < 65536 ? g : 65536);
}

}  // namespace

int quantize(const void* x, int64_t x_stride, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t k, int dtype, int format,
             hipStream_t stream) {
    hipError_t e = hipSuccess;
    by_type(dtype, format, [&](auto t, auto f) {
        using T = decltype(t);
        const int64_t count = rows * (k / kLane);
        e = start(&mx_quantize_kernel<T, decltype(f)::value>, dim3(grid_for(count)), kThreads, 0, stream, 
            static_cast<const typename T::elem*>(x), x_stride, codes, scales, count, (uint32_t)(k / kLane));
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
        e = start(&mx_dequantize_kernel<T, decltype(f)::value>, dim3(grid_for(count)), kThreads, 0, static_cast<hipStream_t>(stream), 
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
    if (rows >= ((int64_t)1 << 31)) return refuse(NQX_ERR_UNSUPPORTED, "%s: too many rows (%lld)", fn, (long long)rows);
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
        e = start(&mx_silu_mul_kernel<T, decltype(f)::value>, dim3(grid_for(count)), kThreads, 0, static_cast<hipStream_t>(stream), 
            static_cast<const E*>(gate), gate_stride, static_cast<const E*>(up), up_stride, codes, scales, count,
            (uint32_t)(k / kLane));
    });
    return hip_status(fn, e);
}
