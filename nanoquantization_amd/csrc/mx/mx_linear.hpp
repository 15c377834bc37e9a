// Launchers of the products of libnq_mx.so; mx_linear.hip chooses among them.
#pragma once

#include "mx_common.hpp"

namespace nqx {

// y [rows, n] = x . w^T + bias; w [n, k / 2] e2m1 and ws [n, k / 32].
struct Product {
    const uint8_t* x;
    const uint8_t* xs;
    const uint8_t* w;
    const uint8_t* ws;
    const void* bias;
    void* y;
    int64_t rows, n, k;
    int dtype, format;
    float* sums;                // what stream_sums_bytes asks for
    const void* raw = nullptr;  // in place of x and xs: x of the call's type, rows raw_stride apart
    int64_t raw_stride = 0;
};

// One matrix instruction: 16 weight rows x 16 rows of x over 128 values (four blocks).  Lane l has row l % 16 and, with
// g = l / 16, block g in e2m1 (16 bytes); in e4m3 the 16 bytes of values 16 g .. and those of 64 + 16 g ...  Its scale byte
// is that of block g for either type, byte BYTE of the word.  The result: column l % 16, weight rows 4 g .. 4 g + 3.
template <int FORMAT, int BYTE = 0>
__device__ __forceinline__ f32x4 mfma(u32x4 w, u32x4 x0, u32x4 x1, f32x4 c, uint32_t w_scale, uint32_t x_scale) {
    const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    const i32x8 b = {(int)x0[0], (int)x0[1], (int)x0[2], (int)x0[3], (int)x1[0], (int)x1[1], (int)x1[2], (int)x1[3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, FORMAT == NQX_FP4 ? 4 : 0, BYTE, (int)w_scale, BYTE, (int)x_scale);
}

// e2m1 with e2m1: 32 weight rows x 32 rows of x over 64 values.  Lane l has row l % 32 and one block; with h = l / 32 the result is
// column l % 32, weight rows 8 q + 4 h .. 8 q + 4 h + 3 in the elements 4 q .. 4 q + 3.  BYTE: which byte of the words holds the scales.
template <int BYTE>
__device__ __forceinline__ f32x16 mfma32(u32x4 w, u32x4 x, f32x16 c, uint32_t w_scale, uint32_t x_scale) {
    const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    const i32x8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 4, 4, BYTE, (int)w_scale, BYTE, (int)x_scale);
}

// V values of a bias from n on, those past the end any; asked for before a kernel's work, not behind it, where a request is a
// microsecond that nothing hides.
template <typename T, int V>
__device__ __forceinline__ void load_bias(float (&b)[V], const typename T::elem* bias, int64_t n, int64_t N) {
    typename T::elem e[V];
    if (n + V <= N) {
        __builtin_memcpy(e, bias + n, sizeof e);     // any address of the type
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] = bias[n + i < N ? n + i : N - 1];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) b[i] = T::to_f32(e[i]);
}
// 4 Q consecutive values of a row of y, columns n and on, of which those below N exist.
template <typename T, int Q>
__device__ __forceinline__ void store_sums(const f32x4 (&v)[Q], typename T::elem* y, int64_t row, int64_t n, int64_t N) {
    typename T::elem* to = y + row * N + n;
    if (n + 4 * Q <= N) {
        // any address of the type
        if constexpr (sizeof(typename T::elem) == 4) {
            __builtin_memcpy(to, v, 16 * Q);
        } else {
            uint32_t w[2 * Q];
#pragma unroll
            for (int q = 0; q < Q; ++q) w[2 * q] = T::pack2(v[q][0], v[q][1]), w[2 * q + 1] = T::pack2(v[q][2], v[q][3]);
            __builtin_memcpy(to, w, 8 * Q);
        }
        return;
    }
#pragma unroll
    for (int r = 0; r < 4 * Q - 1; ++r)
        if (n + r < N) to[r] = T::from_f32(v[r / 4][r % 4]);
}
int skinny_product(const Product& p, hipStream_t stream);       // at most 16 rows of raw x
int64_t skinny_raw_bytes(int64_t rows, int64_t k, int format);
int tiles_product(const Product& p, int tile, hipStream_t stream);
int stream_product(const Product& p, hipStream_t stream);       // at most 128 rows, at most 16 of raw x
bool stream_splits(int64_t rows, int64_t n, int64_t k, int format);
size_t stream_sums_bytes(int64_t rows, int64_t n, int64_t k, int format);
int stream_raw_bytes(int64_t rows, int64_t n, int64_t k, int format);

}  // namespace nqx
