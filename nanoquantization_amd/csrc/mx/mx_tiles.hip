// The product for many rows of x: tiles of TW weight rows x TX rows of x, four waves of a quarter each, on the scaled matrix
// instruction.  A stage is 128 values of k: 64 bytes of a weight row, 64 or 128 of a row of x.  Stages come to LDS by
// load-to-LDS several stages ahead; a wave keeps its weight fragments of a stage in registers, reads those of the next one
// while it multiplies, and the fragments of x two steps ahead of their products.  One barrier a stage: it says that the next
// stage has landed and that the buffer of the last one is free.
#include "../pingpong.hpp"
#include "mx_linear.hpp"

namespace nqx {
namespace {

template <typename T, int FORMAT, int TW, int TX>
struct Tiles {
    static constexpr int kThreads = 256;
    static constexpr int kXB = FORMAT == NQX_FP4 ? 64 : 128;                    // bytes of a row of x in a stage
    static constexpr int kX = TW * 64, kBuf = kX + TX * kXB;                    // [weight rows | x rows]
    static constexpr int kBufs = FORMAT == NQX_FP4 ? 4 : 3;
    static constexpr int kRows = TW + TX;
    static constexpr int kScales = kBufs * kBuf, kSlot = kRows * 16;            // scale bytes of four stages, two slots
    static constexpr int kLds = kScales + 2 * kSlot;
    static constexpr int WT = TW / 32, XT = TX / 32;                            // 16 x 16 tiles of a wave
    static constexpr int kWLoads = TW / 64, kXLoads = TX * kXB / 4096;          // load-to-LDS of a wave and stage, 1 KiB each
    static constexpr int kLoads = kWLoads + kXLoads;
    static constexpr int kRing = 4;
    static_assert(kLds <= 160 * 1024 && kLoads < 16 && XT % kRing == 0 && WT == XT);

    struct Fragment {
        u32x4 lo, hi;       // hi: e4m3 only
        uint32_t scale;
    };
};


template <typename T, int FORMAT, int TW, int TX>
__global__ __launch_bounds__(256, (TW + TX > 256 ? 1 : 2)) void mx_tiles_kernel(
    const uint8_t* __restrict__ x, const uint8_t* __restrict__ xs, const uint8_t* __restrict__ w, const uint8_t* __restrict__ ws,
    const typename T::elem* __restrict__ bias, typename T::elem* __restrict__ y, int rows, int N, int blocks, int x_tiles, int w_tiles) {
    using G = Tiles<T, FORMAT, TW, TX>;
    using Fragment = typename G::Fragment;
    constexpr int WT = G::WT, XT = G::XT;
    extern __shared__ __attribute__((aligned(16))) unsigned char s_mem[];
    int xt, wt;
    if (!awq::xcd_tile(blockIdx.x, x_tiles, w_tiles, xt, wt)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lo = lane & 15, hi = lane >> 4;
    const int wm = wave & 1, wn = wave >> 1;
    const int64_t n0 = (int64_t)wt * TW, m0 = (int64_t)xt * TX;
    const int n_rows = N - n0 < TW ? (int)(N - n0) : TW, m_rows = rows - m0 < TX ? (int)(rows - m0) : TX;
    const uint32_t w_pitch = (uint32_t)blocks * 16, x_pitch = (uint32_t)blocks * (FORMAT == NQX_FP4 ? 16 : 32);
    const uint8_t *wb = w + n0 * w_pitch, *xb = x + m0 * x_pitch, *wsb = ws + n0 * blocks, *xsb = xs + m0 * blocks;
    const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(wb), 0, n_rows * w_pitch, 0x00020000);
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(xb), 0, m_rows * x_pitch, 0x00020000);

    // A load-to-LDS writes 1 KiB in the order of the lanes: 16 rows of 64 bytes, or 8 of 128.  A row's 16-byte pieces are
    // stored at position piece ^ f(row), f = row / 4 % 4 or row / 2 % 8, which spreads the 16 rows of a fragment read over all
    // banks; the swizzle is in the source addresses, four or eight consecutive lanes of which are still one row's.
    uint32_t vw[G::kWLoads], vx[G::kXLoads];
    const auto small_row = [&](int q) { return 16 * (wave + 4 * q) + (lane >> 2); };
    const auto large_row = [&](int q) { return 8 * (wave + 4 * q) + (lane >> 3); };
    const int small_piece = (lane & 3) ^ (lane >> 4), large_piece = (lane & 7) ^ (4 * (wave & 1) + (lane >> 4));
#pragma unroll
    for (int q = 0; q < G::kWLoads; ++q) {
        const int r = small_row(q);
        vw[q] = (uint32_t)(r < n_rows ? r : n_rows - 1) * w_pitch + small_piece * 16;
    }
#pragma unroll
    for (int q = 0; q < G::kXLoads; ++q) {
        const int r = FORMAT == NQX_FP4 ? small_row(q) : large_row(q);
        vx[q] = (uint32_t)(r < m_rows ? r : m_rows - 1) * x_pitch + (FORMAT == NQX_FP4 ? small_piece : large_piece) * 16;
    }
    // Stages: the blocks that do not fill one come first (they need zeros, written by the waves), then the whole ones.
    const int part = blocks & 3, whole = blocks >> 2, first = part ? 1 : 0, stages = whole + first;
    const auto bring = [&](__amdgpu_buffer_rsrc_t r, uint32_t v, int to, int from) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(s_mem + to), 16, v, from, 0, 0);
    };
    const auto load = [&](int t, int at) {          // whole stage t to the buffer at `at`
        const int f = t - first;
#pragma unroll
        for (int q = 0; q < G::kWLoads; ++q) bring(rw, vw[q], at + (wave + 4 * q) * 1024, f * 64);
#pragma unroll
        for (int q = 0; q < G::kXLoads; ++q) bring(rx, vx[q], at + G::kX + (wave + 4 * q) * 1024, f * G::kXB);
    };
    // Scales: 16 bytes of a row are four stages'; a thread brings those of a weight row and of a row of x to registers and,
    // a stage later, to the slot that is free.  The last sixteen are those at the row's end, wherever they start.
    u32x4 sw = {0, 0, 0, 0}, sx = {0, 0, 0, 0};
    const int my_w = (int)threadIdx.x < n_rows ? (int)threadIdx.x : n_rows - 1, my_x = (int)threadIdx.x < m_rows ? (int)threadIdx.x : m_rows - 1;
    const uint8_t *swp = wsb + (int64_t)my_w * blocks, *sxp = xsb + (int64_t)my_x * blocks;
    const auto start_of = [&](int u) { return 16 * u + 16 <= blocks ? 16 * u : blocks - 16; };
    const auto load_scales = [&](int u) {
        const int at = start_of(u);
        __builtin_memcpy(&sw, swp + at, 16);
        __builtin_memcpy(&sx, sxp + at, 16);
    };
    const auto store_scales = [&](int slot) {
        unsigned char* s = s_mem + G::kScales + slot * G::kSlot;
        if ((int)threadIdx.x < TW) *reinterpret_cast<u32x4*>(s + threadIdx.x * 16) = sw;
        if ((int)threadIdx.x < TX) *reinterpret_cast<u32x4*>(s + (TW + threadIdx.x) * 16) = sx;
    };
    const auto few_scales = [&](int from, int count, uint32_t (&w4)[4], const uint8_t* p) {     // bytes, the rest 127
        for (int i = 0; i < 4; ++i) w4[i] = 0x7F7F7F7Fu;
        for (int i = 0; i < count; ++i) w4[i >> 2] = (w4[i >> 2] & ~(0xFFu << (8 * (i & 3)))) | (uint32_t)p[from + i] << (8 * (i & 3));
    };
    const auto byte_scales = [&](int from, int count) {
        uint32_t a[4], b[4];
        few_scales(from, count, a, swp);
        few_scales(from, count, b, sxp);
        sw = u32x4{a[0], a[1], a[2], a[3]}, sx = u32x4{b[0], b[1], b[2], b[3]};
    };

    const int w_at = (wm * (TW / 2) + lo) * 64 + ((hi ^ (lo >> 2)) & 3) * 16;
    const int x_at = FORMAT == NQX_FP4 ? G::kX + (wn * (TX / 2) + lo) * 64 + ((hi ^ (lo >> 2)) & 3) * 16
                                       : G::kX + (wn * (TX / 2) + lo) * 128 + ((hi ^ (lo >> 1)) & 7) * 16;
    const int ws_at = G::kScales + (wm * (TW / 2) + lo) * 16 + hi, xs_at = G::kScales + (TW + wn * (TX / 2) + lo) * 16 + hi;
    const auto read_w = [&](Fragment& f, int at, int s, int i) {
        f.lo = *reinterpret_cast<const u32x4*>(s_mem + at + w_at + i * 1024);
        f.scale = s_mem[ws_at + s + i * 256];
    };
    const auto read_x = [&](Fragment& f, int at, int s, int j) {
        const int p = at + x_at + j * 16 * G::kXB;
        f.lo = *reinterpret_cast<const u32x4*>(s_mem + p);
        if constexpr (FORMAT == NQX_FP8) f.hi = *reinterpret_cast<const u32x4*>(s_mem + (p ^ 64));
        f.scale = s_mem[xs_at + s + j * 256];
    };
    // Where the scales of stage t are, from those of stage 0 of slot 0 on.
    const auto scales_of = [&](int t) {
        const int f = t - first, u = f >> 2;
        return f < 0 ? G::kSlot : (u & 1) * G::kSlot + 4 * f - (blocks < 16 ? 0 : start_of(u));
    };

    f32x4 acc[WT][XT];
#pragma unroll
    for (int i = 0; i < WT; ++i)
#pragma unroll
        for (int j = 0; j < XT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // ---- before the first stage ----
    if (whole) {
        if (blocks < 16) byte_scales(0, blocks);
        else load_scales(0);
        store_scales(0);
    }
    if (part) {
        byte_scales(4 * whole, part);
        store_scales(1);
#pragma unroll
        for (int q = 0; q < G::kWLoads; ++q) {
            u32x4 v = {0, 0, 0, 0};
            if (small_piece < part) v = *reinterpret_cast<const u32x4*>(wb + vw[q] + whole * 64);
            *reinterpret_cast<u32x4*>(s_mem + (wave + 4 * q) * 1024 + lane * 16) = v;
        }
#pragma unroll
        for (int q = 0; q < G::kXLoads; ++q) {
            u32x4 v = {0, 0, 0, 0};
            if ((FORMAT == NQX_FP4 ? small_piece : large_piece / 2) < part) v = *reinterpret_cast<const u32x4*>(xb + vx[q] + whole * G::kXB);
            *reinterpret_cast<u32x4*>(s_mem + G::kX + (wave + 4 * q) * 1024 + lane * 16) = v;
        }
    }
    int at = 0;                                      // buffer of stage t, of stage t + 1, and the one that stage t - 1 had
    int next = G::kBuf, free_at = (G::kBufs - 1) * G::kBuf;
#pragma unroll
    for (int t = 0; t < G::kBufs - 1; ++t)
        if (t >= first && t < stages) load(t, t * G::kBuf);
    __builtin_amdgcn_s_waitcnt(0x0070);              // everything so far is there: vmcnt(0), lgkmcnt(0)
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);

    Fragment a0[WT], a1[WT], b[G::kRing];
    {
        const int s = scales_of(0);
#pragma unroll
        for (int i = 0; i < WT; ++i) read_w(a0[i], at, s, i);
        read_x(b[0], at, s, 0), read_x(b[1], at, s, 1);
    }
    const auto stage = [&](int t, Fragment (&a)[WT], Fragment (&an)[WT]) {
        // the next stage has landed: at most those asked for after it, a stage ago, are on their way
        if (t > 0) {
            if (G::kBufs == 4 && t + 2 < stages) __builtin_amdgcn_s_waitcnt(0x0070 | G::kLoads);    // vmcnt(kLoads) lgkmcnt(0)
            else __builtin_amdgcn_s_waitcnt(0x0070);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
        }
        const int f = t - first;
        if (f >= 0) {
            const int u = (f >> 2) + 1;
            if ((f & 3) == 0 && 4 * u < whole) load_scales(u);
            if ((f & 3) == 1 && 4 * u < whole) store_scales(u & 1);
        }
        if (t + G::kBufs - 1 < stages) load(t + G::kBufs - 1, free_at);
        const int s = scales_of(t), sn = scales_of(t + 1 < stages ? t + 1 : t);
#pragma unroll
        for (int j = 0; j < XT; ++j) {
            if (j + 2 < XT) read_x(b[(j + 2) % G::kRing], at, s, j + 2);
            else read_x(b[(j + 2) % G::kRing], next, sn, j + 2 - XT);
            read_w(an[j], next, sn, j);
#pragma unroll
            for (int i = 0; i < WT; ++i)
                acc[i][j] = mfma<FORMAT>(a[i].lo, b[j % G::kRing].lo, b[j % G::kRing].hi, acc[i][j], a[i].scale, b[j % G::kRing].scale);
            __builtin_amdgcn_sched_barrier(0);
        }
        free_at = at, at = next, next = next == (G::kBufs - 1) * G::kBuf ? 0 : next + G::kBuf;
    };
    int t = 0;
#pragma unroll 1
    for (; t + 1 < stages; t += 2) {
        stage(t, a0, a1);
        stage(t + 1, a1, a0);
    }
    if (t < stages) stage(t, a0, a1);

#pragma unroll
    for (int j = 0; j < XT; ++j)
#pragma unroll
        for (int i = 0; i < WT; ++i) {
            const int64_t row = m0 + wn * (TX / 2) + 16 * j + lo, n = n0 + wm * (TW / 2) + 16 * i + 4 * hi;
            if (row < rows && n < N) store_sums<T>(acc[i][j], y, bias, row, n, N);
        }
}

template <typename T, int FORMAT, int S>
hipError_t launch(const Product& p, hipStream_t stream) {
    using G = Tiles<T, FORMAT, S, S>;
    using E = typename T::elem;
    const int x_tiles = (int)cdiv(p.rows, S), w_tiles = (int)cdiv(p.n, S);
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&mx_tiles_kernel<T, FORMAT, S, S>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, G::kLds);
    if (e != hipSuccess) return e;
    const unsigned grid = (unsigned)(cdiv((int64_t)x_tiles * w_tiles, 8) * 8);
    mx_tiles_kernel<T, FORMAT, S, S><<<grid, G::kThreads, G::kLds, stream>>>(
        p.x, p.xs, p.w, p.ws, static_cast<const E*>(p.bias), static_cast<E*>(p.y), (int)p.rows, (int)p.n, (int)(p.k / kBlock), x_tiles,
        w_tiles);
    return hipGetLastError();
}

}  // namespace

int tiles_product(const Product& p, int tile, hipStream_t stream) {
    hipError_t e = hipSuccess;
    by_type(p.dtype, p.format, [&](auto t, auto f) {
        using T = decltype(t);
        constexpr int F = decltype(f)::value;
        e = tile == 256 ? launch<T, F, 256>(p, stream) : launch<T, F, 128>(p, stream);
    });
    return e == hipSuccess ? NQX_OK : refuse(NQX_ERR_HIP, "mx_tiles_kernel: HIP error %d (%s)", (int)e, hipGetErrorString(e));
}

}  // namespace nqx
