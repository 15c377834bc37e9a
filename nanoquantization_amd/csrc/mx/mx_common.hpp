// What the kernels of microscaled formats share (libnq_mx.so): element types, the arithmetic of a block, error plumbing.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>
#include <tuple>

#include "../../../include/nq_mx_ops.h"

namespace nqx {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kBlock = 32;      // values of a block
constexpr int kLane = 8;        // values that a lane of the row kernels holds: four lanes a block

struct F16 {
    using elem = uint16_t;
    static constexpr int id = NQX_F16;
    static __device__ __forceinline__ float to_f32(uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }
    static __device__ __forceinline__ uint16_t from_f32(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) {
        return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
    }
};
struct BF16 {
    using elem = uint16_t;
    static constexpr int id = NQX_BF16;
    static __device__ __forceinline__ float to_f32(uint16_t b) { return __builtin_bit_cast(float, (uint32_t)b << 16); }
    static __device__ __forceinline__ uint16_t from_f32(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) {
        return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
    }
};
struct F32 {
    using elem = float;
    static constexpr int id = NQX_F32;
    static __device__ __forceinline__ float to_f32(float f) { return f; }
    static __device__ __forceinline__ float from_f32(float f) { return f; }
};

// (By value: a bit_cast of a vector's element takes the vector's first.)
template <typename V>
__device__ __forceinline__ V as(uint32_t bits) {
    return __builtin_bit_cast(V, bits);
}

// Eight consecutive elements, 16-byte accesses.
template <typename T>
__device__ __forceinline__ void load8(const typename T::elem* p, float (&v)[8]) {
    if constexpr (sizeof(typename T::elem) == 4) {
        const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    } else {
        const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = w[i];
            v[2 * i] = T::to_f32((uint16_t)(u & 0xFFFFu)), v[2 * i + 1] = T::to_f32((uint16_t)(u >> 16));
        }
    }
}
template <typename T>
__device__ __forceinline__ void store8(typename T::elem* p, const float (&v)[8]) {
    if constexpr (sizeof(typename T::elem) == 4) {
        reinterpret_cast<f32x4*>(p)[0] = f32x4{v[0], v[1], v[2], v[3]};
        reinterpret_cast<f32x4*>(p)[1] = f32x4{v[4], v[5], v[6], v[7]};
    } else {
        *reinterpret_cast<u32x4*>(p) = u32x4{T::pack2(v[0], v[1]), T::pack2(v[2], v[3]), T::pack2(v[4], v[5]), T::pack2(v[6], v[7])};
    }
}

// 2^(byte - 127) as fp32: the byte is the float's exponent field, but for 0 (2^-127, a subnormal) and 255 (NaN).
__device__ __forceinline__ float power(uint32_t byte) {
    const uint32_t bits = byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23;
    return __builtin_bit_cast(float, bits);
}
// The scale byte of a block whose largest magnitude has these bits (as integers they are ordered like the magnitudes, NaN
// and infinity on top).  The largest element is 1.5 * 2^2 (e2m1) or 1.75 * 2^8 (e4m3), and a magnitude of 1.75 * 2^n and
// above, or of more than 1.8125 * 2^n, rounds past it: the addition carries exactly those into the exponent field.
template <int FORMAT>
__device__ __forceinline__ uint32_t scale_byte(uint32_t bits) {
    const int byte = (int)((bits + (FORMAT == NQX_FP4 ? 0x200000u : 0x17FFFFu)) >> 23) - (FORMAT == NQX_FP4 ? 2 : 8);
    return bits >= 0x7F800000u ? 255u : (uint32_t)(byte < 0 ? 0 : byte);
}
__device__ __forceinline__ uint32_t magnitude_bits(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu);
    return m;
}
// The largest of the four lanes of a block (an aligned group), in each of them.
__device__ __forceinline__ uint32_t max_of_block(uint32_t m) {
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, true));   // lanes 1 0 3 2
    return max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, true));  // lanes 2 3 0 1
}
// Codes of eight values: four bytes of e2m1 (.x) or eight of e4m3.  The conversion divides by the power of two exactly and
// rounds once, to nearest with ties to even; no value is past the largest element's rounding range, which e4m3 would turn
// into a NaN.
template <int FORMAT>
__device__ __forceinline__ u32x2 encode8(const float (&v)[8], uint32_t byte) {
    if (byte == 255) return u32x2{0u, 0u};
    const float scale = power(byte);
    if constexpr (FORMAT == NQX_FP4) {
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
        return u32x2{w, 0u};
    } else {
        i16x2 a = {0, 0}, b = {0, 0};
        a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[0], v[1], scale, false);
        a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[2], v[3], scale, true);
        b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[4], v[5], scale, false);
        b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[6], v[7], scale, true);
        return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
    }
}
// Eight 16-bit values as they are in memory: magnitudes two at a time, and conversions that take the pairs.
template <typename T>
__device__ __forceinline__ uint32_t magnitude_bits(u32x4 w) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 m = __builtin_bit_cast(u16x2, w[0] & 0x7FFF7FFFu);
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu));
    return __builtin_bit_cast(uint32_t, T::to_f32(m[0] > m[1] ? m[0] : m[1]));
}
template <typename T, int FORMAT>
__device__ __forceinline__ u32x2 encode8(u32x4 w, uint32_t byte) {
    if (byte == 255) return u32x2{0u, 0u};
    const float scale = power(byte);
    if constexpr (FORMAT == NQX_FP4) {
        uint32_t c = 0;
        if constexpr (T::id == NQX_BF16) {
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, as<bf16x2>(w[0]), scale, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, as<bf16x2>(w[1]), scale, 1);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, as<bf16x2>(w[2]), scale, 2);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, as<bf16x2>(w[3]), scale, 3);
        } else {
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, as<f16x2>(w[0]), scale, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, as<f16x2>(w[1]), scale, 1);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, as<f16x2>(w[2]), scale, 2);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, as<f16x2>(w[3]), scale, 3);
        }
        return u32x2{c, 0u};
    } else {
        i16x2 a = {0, 0}, b = {0, 0};
        if constexpr (T::id == NQX_BF16) {
            a = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(a, as<bf16x2>(w[0]), scale, false);
            a = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(a, as<bf16x2>(w[1]), scale, true);
            b = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(b, as<bf16x2>(w[2]), scale, false);
            b = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(b, as<bf16x2>(w[3]), scale, true);
        } else {
            a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(a, as<f16x2>(w[0]), scale, false);
            a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(a, as<f16x2>(w[1]), scale, true);
            b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(b, as<f16x2>(w[2]), scale, false);
            b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(b, as<f16x2>(w[3]), scale, true);
        }
        return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
    }
}
// One lane's part of a quantised row: its codes and, of the four lanes of a block, the first one's scale, number `at` of the
// tensor's eights.
template <int FORMAT>
__device__ __forceinline__ void put8(u32x2 code, uint32_t byte, uint8_t* codes, uint8_t* scales, int64_t at) {
    if constexpr (FORMAT == NQX_FP4) reinterpret_cast<uint32_t*>(codes)[at] = code.x;
    else reinterpret_cast<u32x2*>(codes)[at] = code;
    if ((at & 3) == 0) scales[at >> 2] = (uint8_t)byte;
}
// All four lanes of a block call it.
template <int FORMAT>
__device__ __forceinline__ void quantize8(const float (&v)[8], uint8_t* codes, uint8_t* scales, int64_t at) {
    const uint32_t byte = scale_byte<FORMAT>(max_of_block(magnitude_bits(v)));
    put8<FORMAT>(encode8<FORMAT>(v, byte), byte, codes, scales, at);
}
// Eight values at p, quantised: of 16-bit types without a detour over fp32, the same codes.
template <typename T, int FORMAT>
struct Eight {
    u32x4 w[T::id == NQX_F32 ? 2 : 1];
    __device__ __forceinline__ void load(const typename T::elem* p) {
        w[0] = reinterpret_cast<const u32x4*>(p)[0];
        if constexpr (T::id == NQX_F32) w[1] = reinterpret_cast<const u32x4*>(p)[1];
    }
    __device__ __forceinline__ void clear() {
        w[0] = u32x4{0u, 0u, 0u, 0u};
        if constexpr (T::id == NQX_F32) w[1] = w[0];
    }
    __device__ __forceinline__ void floats(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (T::id == NQX_F32) {
                v[i] = as<float>(w[0][i]), v[4 + i] = as<float>(w[1][i]);
            } else {
                const uint32_t u = w[0][i];
                v[2 * i] = T::to_f32((uint16_t)(u & 0xFFFFu)), v[2 * i + 1] = T::to_f32((uint16_t)(u >> 16));
            }
        }
    }
    // the codes; `byte`: the scale
    __device__ __forceinline__ u32x2 encode(uint32_t& byte) const {
        if constexpr (T::id == NQX_F32) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = as<float>(w[i / 4][i % 4]);
            byte = scale_byte<FORMAT>(max_of_block(magnitude_bits(v)));
            return encode8<FORMAT>(v, byte);
        } else {
            byte = scale_byte<FORMAT>(max_of_block(magnitude_bits<T>(w[0])));
            return encode8<T, FORMAT>(w[0], byte);
        }
    }
};

// ---- host ----------------------------------------------------------------------------------------------------------------
int refuse(int status, const char* fmt, ...);
int hip_status(const char* fn, hipError_t e);

// Launches a kernel; what an earlier call of anybody's has left behind is not taken for this one's error.
template <typename... P, typename... A>
static inline hipError_t start(void (*kernel)(P...), dim3 grid, unsigned threads, size_t lds, hipStream_t stream, A... args) {
    std::tuple<P...> held(args...);
    return std::apply([&](auto&... a) {
        void* at[] = {const_cast<void*>(static_cast<const void*>(&a))...};
        return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(threads), at, lds, stream);
    }, held);
}
// More than 64 KiB of LDS for a kernel, once for each device.
template <auto KERNEL>
static inline hipError_t allow_lds(int bytes) {
    static std::atomic<uint64_t> done{0};
    int device = 0;
    if (const hipError_t e = hipGetDevice(&device); e != hipSuccess) return e;
    const uint64_t bit = 1ull << (device & 63);
    if (done.load(std::memory_order_relaxed) & bit) return hipSuccess;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}
static inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
static inline int64_t elem_bytes(int dtype) { return dtype == NQX_F32 ? 4 : 2; }
static inline int64_t code_bytes(int64_t k, int format) { return format == NQX_FP4 ? k / 2 : k; }

// Calls f with the types of a call as arguments: F16(), BF16() or F32(), and the format as an integral constant.
template <int V>
struct Const {
    static constexpr int value = V;
};
template <typename F>
static inline void by_type(int dtype, int format, F&& f) {
    const auto with = [&](auto t) {
        if (format == NQX_FP4) f(t, Const<NQX_FP4>());
        else f(t, Const<NQX_FP8>());
    };
    if (dtype == NQX_F16) with(F16());
    else if (dtype == NQX_BF16) with(BF16());
    else with(F32());
}

// Sizes and types that every entry point shares: rows may be 0, then there is nothing to do.
int check_types(const char* fn, int64_t rows, int64_t k, int dtype, int format);
int check_rows(const char* fn, const char* what, const void* p, int64_t stride, int64_t k, int dtype);
int quantize(const void* x, int64_t x_stride, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t k, int dtype, int format,
             hipStream_t stream);

}  // namespace nqx
