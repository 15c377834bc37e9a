// The product for few rows of x: the packed weight streams from memory once, 0.53 bytes a value, and everything else hides
// behind it.  A workgroup owns 16 * NT weight rows and 16 * MT rows of x; its eight waves share out k in units of 512 values
// (256 bytes of a weight row) and their sums meet in LDS, always in the order of the waves.  Operands go from memory
// straight into the registers that the matrix instruction reads: a lane's 16 bytes are its block.
#include "mx_linear.hpp"

namespace nqx {
namespace {

constexpr int kWaves = 8;
constexpr int kUnit = 16;       // blocks

template <typename T, int FORMAT, int MT, int NT>
__global__ __launch_bounds__(64 * kWaves) void mx_skinny_kernel(const uint8_t* __restrict__ x, const uint8_t* __restrict__ xs,
                                                                const uint8_t* __restrict__ w, const uint8_t* __restrict__ ws,
                                                                const typename T::elem* __restrict__ bias,
                                                                typename T::elem* __restrict__ y, int64_t rows, int64_t N,
                                                                int blocks) {
    __shared__ f32x4 s_acc[kWaves][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lo = lane & 15, hi = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * NT), m0 = (int64_t)blockIdx.y * (16 * MT);
    const int64_t w_pitch = (int64_t)blocks * 16, x_pitch = (int64_t)blocks * (FORMAT == NQX_FP4 ? 16 : 32);
    // rows past the end: the last row again, of which nothing is stored
    const uint8_t *wp[NT], *wsp[NT], *xp[MT], *xsp[MT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int64_t r = n0 + 16 * i + lo < N ? n0 + 16 * i + lo : N - 1;
        wp[i] = w + r * w_pitch, wsp[i] = ws + r * blocks;
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int64_t r = m0 + 16 * j + lo < rows ? m0 + 16 * j + lo : rows - 1;
        xp[j] = x + r * x_pitch, xsp[j] = xs + r * blocks;
    }
    f32x4 acc[MT][NT];
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};

    // four matrix steps from block b0 on; of a unit that the row ends in, the blocks behind the end count as zeros
    const auto unit = [&](int b0, auto whole) {
        constexpr bool kWhole = decltype(whole)::value != 0;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int b = b0 + 4 * s + hi;
            const bool in = kWhole || b < blocks;
            u32x4 wv[NT], x0[MT], x1[MT];
            uint32_t wsv[NT], xsv[MT];
            const u32x4 none = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                wv[i] = in ? *reinterpret_cast<const u32x4*>(wp[i] + (int64_t)b * 16) : none;
                wsv[i] = in ? wsp[i][b] : 127u;
            }
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                xsv[j] = in ? xsp[j][b] : 127u;
                if constexpr (FORMAT == NQX_FP4) {
                    x0[j] = x1[j] = in ? *reinterpret_cast<const u32x4*>(xp[j] + (int64_t)b * 16) : none;
                } else {
                    const int at = (b0 + 4 * s) * 32 + 16 * hi;
                    x0[j] = kWhole || at < blocks * 32 ? *reinterpret_cast<const u32x4*>(xp[j] + at) : none;
                    x1[j] = kWhole || at + 64 < blocks * 32 ? *reinterpret_cast<const u32x4*>(xp[j] + at + 64) : none;
                }
            }
#pragma unroll
            for (int j = 0; j < MT; ++j)
#pragma unroll
                for (int i = 0; i < NT; ++i) acc[j][i] = mfma<FORMAT>(wv[i], x0[j], x1[j], acc[j][i], wsv[i], xsv[j]);
        }
    };
    int b0 = wave * kUnit;
    for (; b0 + kUnit <= blocks; b0 += kWaves * kUnit) unit(b0, Const<1>());
    if (b0 < blocks) unit(b0, Const<0>());

#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int i = 0; i < NT; ++i) s_acc[wave][j * NT + i][lane] = acc[j][i];
    __syncthreads();
    for (int t = wave; t < MT * NT; t += kWaves) {
        f32x4 sum = s_acc[0][t][lane];
#pragma unroll
        for (int v = 1; v < kWaves; ++v) sum += s_acc[v][t][lane];
        const int64_t row = m0 + 16 * (t / NT) + lo, n = n0 + 16 * (t % NT) + 4 * hi;
        if (row < rows && n < N) store_sums<T>(sum, y, bias, row, n, N);
    }
}

}  // namespace

int skinny_product(const Product& p, hipStream_t stream) {
    by_type(p.dtype, p.format, [&](auto t, auto f) {
        using T = decltype(t);
        using E = typename T::elem;
        const auto with = [&](auto mt, auto nt) {
            constexpr int MT = decltype(mt)::value, NT = decltype(nt)::value;
            const dim3 grid((unsigned)cdiv(p.n, 16 * NT), (unsigned)cdiv(p.rows, 16 * MT));
            mx_skinny_kernel<T, decltype(f)::value, MT, NT><<<grid, 64 * kWaves, 0, stream>>>(
                p.x, p.xs, p.w, p.ws, static_cast<const E*>(p.bias), static_cast<E*>(p.y), p.rows, p.n, (int)(p.k / kBlock));
        };
        if (p.rows <= 16) with(Const<1>(), Const<1>());
        else with(Const<2>(), Const<2>());
    });
    return hip_status("mx_skinny_kernel");
}

}  // namespace nqx
