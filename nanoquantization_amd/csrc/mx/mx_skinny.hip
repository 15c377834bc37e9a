// The product for few rows of x and a weight that is read in a few microseconds, where latency counts: one launch, a workgroup for
// every 16 weight rows, its eight waves share out k in steps of 128 values and their sums meet in LDS, always in the order of the
// waves.  Operands go from memory straight into the registers that the matrix instruction reads: a lane's 16 bytes are its block.
//
// With RAW x comes as it is: a workgroup asks for its first weights, quantises all of x into LDS and multiplies from there.
#include "mx_linear.hpp"

namespace nqx {
namespace {

constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kAhead = 4;       // steps of a wave whose weights are on their way at once

template <typename T, int FORMAT, int MT, bool RAW>
__global__ __launch_bounds__(kThreads) void mx_skinny_kernel(const void* __restrict__ x, int64_t x_stride, const uint8_t* __restrict__ xs,
                                                             const uint8_t* __restrict__ w, const uint8_t* __restrict__ ws,
                                                             const typename T::elem* __restrict__ bias,
                                                             typename T::elem* __restrict__ y, int64_t rows, int64_t N, int blocks) {
    constexpr bool kFour = FORMAT == NQX_FP4;
    constexpr int kBytes = kFour ? 16 : 32;          // of a block of x
    __shared__ f32x4 s_acc[kWaves][MT][64];
    extern __shared__ __attribute__((aligned(16))) unsigned char s_x[];     // RAW: codes of all rows, a row's in steps, then scales
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lo = lane & 15, hi = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * (16 * MT);
    // rows past the end: the last row again, of which nothing is stored
    const int64_t n = n0 + lo < N ? n0 + lo : N - 1;
    const uint8_t *wp = w + n * blocks * 16, *wsp = ws + n * blocks;
    const uint8_t *xp[MT], *xsp[MT];
    const int steps = (blocks + 3) >> 2, r_bytes = steps * 4 * kBytes;
    const unsigned char* s_xs = s_x + (RAW ? (int)rows * r_bytes : 0);
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int64_t r = m0 + 16 * j + lo < rows ? m0 + 16 * j + lo : rows - 1;
        if constexpr (RAW) xp[j] = s_x + r * r_bytes, xsp[j] = s_xs + r * steps * 4;
        else xp[j] = static_cast<const uint8_t*>(x) + r * blocks * kBytes, xsp[j] = xs + r * blocks;
    }
    f32x4 acc[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // kAhead steps of the wave from step s0 on; blocks past the end have zeros for codes and the scale 2^0
    u32x4 wv[kAhead];
    uint32_t wsv[kAhead];
    const auto ask = [&](int s0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int b = 4 * (s0 + u * kWaves) + hi;
            wv[u] = u32x4{0u, 0u, 0u, 0u}, wsv[u] = 127u;
            if (b < blocks) wv[u] = *reinterpret_cast<const u32x4*>(wp + (int64_t)b * 16), wsv[u] = wsp[b];
        }
    };
    ask(wave);
    float b[4] = {};
    if (bias && wave < MT) load_bias<T>(b, bias, n0 + 4 * hi, N);
    if constexpr (RAW) {
        using E = typename T::elem;
        const int per_row = steps * 16;              // eights
        for (int i = threadIdx.x; i < (int)rows * per_row; i += kThreads) {
            const int r = i / per_row, e = i - r * per_row;
            Eight<T, FORMAT> v;
            v.clear();
            if (e < blocks * 4) v.load(static_cast<const E*>(x) + r * x_stride + e * 8);
            uint32_t byte;
            const u32x2 code = v.encode(byte);
            if constexpr (kFour) *reinterpret_cast<uint32_t*>(s_x + r * r_bytes + e * 4) = code.x;
            else *reinterpret_cast<u32x2*>(s_x + r * r_bytes + e * 8) = code;
            if ((e & 3) == 0) s_x[(int)rows * r_bytes + r * steps * 4 + (e >> 2)] = (unsigned char)byte;
        }
        __syncthreads();
    }
#pragma unroll 1
    for (int s0 = wave; s0 < steps; s0 += kAhead * kWaves) {
        if (s0 != wave) ask(s0);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int s = s0 + u * kWaves, b = 4 * s + hi;
            if (s >= steps) break;
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                const u32x4 none = {0u, 0u, 0u, 0u};
                // RAW: all blocks of a step are there, zeros behind the end
                const bool in = RAW || b < blocks;
                const uint32_t xsv = in ? xsp[j][b] : 127u;
                u32x4 x0, x1;
                if constexpr (kFour) {
                    x0 = x1 = in ? *reinterpret_cast<const u32x4*>(xp[j] + (int64_t)b * 16) : none;
                } else {
                    const int at = s * 128 + 16 * hi;
                    x0 = RAW || at < blocks * 32 ? *reinterpret_cast<const u32x4*>(xp[j] + at) : none;
                    x1 = RAW || at + 64 < blocks * 32 ? *reinterpret_cast<const u32x4*>(xp[j] + at + 64) : none;
                }
                acc[j] = mfma<FORMAT>(wv[u], x0, x1, acc[j], wsv[u], xsv);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) s_acc[wave][j][lane] = acc[j];
    __syncthreads();
    if (wave < MT) {
        f32x4 sum[1] = {s_acc[0][wave][lane]};
#pragma unroll
        for (int v = 1; v < kWaves; ++v) sum[0] += s_acc[v][wave][lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[0][i] += b[i];
        const int64_t row = m0 + 16 * wave + lo, at = n0 + 4 * hi;
        if (row < rows && at < N) store_sums<T>(sum, y, row, at, N);
    }
}

template <typename T, int FORMAT, int MT, bool RAW>
hipError_t launch(const Product& p, hipStream_t stream) {
    using E = typename T::elem;
    const dim3 grid((unsigned)cdiv(p.n, 16), (unsigned)cdiv(p.rows, 16 * MT));
    const size_t lds = RAW ? (size_t)skinny_raw_bytes(p.rows, p.k, FORMAT) : 0;
    return start(&mx_skinny_kernel<T, FORMAT, MT, RAW>, grid, kThreads, lds, stream, RAW ? p.raw : p.x, p.raw_stride, p.xs, p.w, p.ws,
                 static_cast<const E*>(p.bias), static_cast<E*>(p.y), p.rows, p.n, (int)(p.k / kBlock));
}

}  // namespace

int skinny_product(const Product& p, hipStream_t stream) {
    hipError_t e = hipSuccess;
    by_type(p.dtype, p.format, [&](auto t, auto f) {
        using T = decltype(t);
        constexpr int F = decltype(f)::value;
        if (p.raw) e = launch<T, F, 1, true>(p, stream);
        else if (p.rows <= 16) e = launch<T, F, 1, false>(p, stream);
        else e = launch<T, F, 2, false>(p, stream);
    });
    return hip_status("mx_skinny_kernel", e);
}

// x of a raw product in LDS: codes of whole steps, and their scales
int64_t skinny_raw_bytes(int64_t rows, int64_t k, int format) {
    return rows * cdiv(k, 128) * ((format == NQX_FP4 ? 64 : 128) + 4);
}

}  // namespace nqx
