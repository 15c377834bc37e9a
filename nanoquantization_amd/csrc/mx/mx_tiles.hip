// The product for many rows of x: square tiles, four waves of a quarter each, on the scaled matrix instruction.
//
// Operands come to LDS by load-to-LDS in chunks of 256 values of k: 128 bytes of an e2m1 row, a whole line, or twice 128 bytes of
// an e4m3 one.  (What feeds a tile is the L2, and it takes requests, not bytes: with 64 bytes of a row at a time 8192 x 8192 x 8192
// in 4 bits was 334 us, 246 without a matrix instruction.)  Two chunks are in LDS.  A wave reads the fragments of a step while the
// matrix cores have the one before, so at a chunk's last step nobody needs its buffer any more: there is the one barrier of a
// chunk, which also says that the next one has landed, and behind it the requests for the chunk after that go out, over half a
// chunk's products (over three quarters of them 8192 cubed takes 289 us instead of 277, in 8 bits 433 and 425: the last ones are
// waited for).
#include "../pingpong.hpp"
#include "mx_linear.hpp"

namespace nqx {
namespace {

// What the matrix instruction takes at once.  e2m1 on both sides runs on 32 x 32 x 64 (a loop of nothing else reaches 6.4
// PFLOP/s, one of 16 x 16 x 128 5.1); e4m3 with e2m1 on 16 x 16 x 128 (4.0 to 4.2, by the GPU, and 3.5 to 3.9 on 32 x 32 x 64).
template <int FORMAT>
struct Shape {
    static constexpr int kRows = 16;
    typedef f32x4 Sums;
};
template <>
struct Shape<NQX_FP4> {
    static constexpr int kRows = 32;
    typedef f32x16 Sums;
};

template <int FORMAT, int S>
struct Tiles {
    static constexpr int kThreads = 256;
    static constexpr int kPart = S * 128;               // 128 bytes of every row of an operand
    // [two chunks of the weight | two of x (e2m1), or the two halves of one (e4m3) | two slots of scales, 32 bytes a row: four chunks]
    static constexpr int kX = 2 * kPart, kScales = 4 * kPart, kSlot = 2 * S * 32;
    static constexpr int kLds = kScales + 2 * kSlot;
    static constexpr int R = Shape<FORMAT>::kRows, WT = S / 2 / R, XT = S / 2 / R;       // fragments of a wave
    static constexpr int kLoads = S / 32;               // load-to-LDS of a wave for a part, 1 KiB each
    static_assert(kLds <= 160 * 1024, "");
};

template <typename T, int FORMAT, int S, bool BIAS>
__global__ __launch_bounds__(256, (S == 256 ? 1 : 2)) void mx_tiles_kernel(
    const uint8_t* __restrict__ x, const uint8_t* __restrict__ xs, const uint8_t* __restrict__ w, const uint8_t* __restrict__ ws,
    const typename T::elem* __restrict__ bias, typename T::elem* __restrict__ y, int rows, int N, int blocks, int words, int x_tiles,
    int w_tiles) {
    using G = Tiles<FORMAT, S>;
    using Sums = typename Shape<FORMAT>::Sums;
    constexpr int WT = G::WT, XT = G::XT, R = G::R, TW = S, TX = S;
    constexpr bool kFour = FORMAT == NQX_FP4;
    extern __shared__ __attribute__((aligned(16))) unsigned char s_mem[];
    int xt, wt;
    if (!awq::xcd_tile(blockIdx.x, x_tiles, w_tiles, xt, wt)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = lane & (R - 1), part_of = lane / R;   // of a fragment
    const int wm = wave & 1, wn = wave >> 1;
    const int64_t n0 = (int64_t)wt * TW, m0 = (int64_t)xt * TX;
    const int n_rows = N - n0 < TW ? (int)(N - n0) : TW, m_rows = rows - m0 < TX ? (int)(rows - m0) : TX;
    const uint32_t w_pitch = (uint32_t)blocks * 16, x_pitch = (uint32_t)blocks * (kFour ? 16 : 32);
    const uint8_t *wb = w + n0 * w_pitch, *xb = x + m0 * x_pitch, *wsb = ws + n0 * blocks, *xsb = xs + m0 * blocks;

    // A load-to-LDS writes 1 KiB in the order of the lanes: eight rows of 128 bytes.  A row's 16-byte pieces are stored at position
    // piece ^ (row / 2 % 8), which spreads the rows of a fragment read over all banks; the swizzle is in the source addresses,
    // eight consecutive lanes of which are still one row's.  Rows past the end: the last row again, of which nothing is stored.
    uint32_t vw[G::kLoads], vx[G::kLoads];
    const int piece = (lane & 7) ^ (4 * (wave & 1) + (lane >> 4));
#pragma unroll
    for (int q = 0; q < G::kLoads; ++q) {
        const int r = 8 * (wave + 4 * q) + (lane >> 3);
        vw[q] = (uint32_t)(r < n_rows ? r : n_rows - 1) * w_pitch + piece * 16;
        vx[q] = (uint32_t)(r < m_rows ? r : m_rows - 1) * x_pitch + piece * 16;
    }
    // Chunks: the blocks that do not fill one come first (they need zeros, written by the waves), then the whole ones.
    const int part = blocks & 7, whole = blocks >> 3, first = part ? 1 : 0, chunks = whole + first;
    const auto bring = [&](__amdgpu_buffer_rsrc_t r, uint32_t v, int to, int from) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(s_mem + to), 16, v, from, 0, 0);
    };
    const auto buffer = [](const uint8_t* p, uint32_t bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, bytes, 0x00020000);
    };
    // Load q of a chunk's weight, and of x: e2m1 a chunk's, e4m3 those of half a chunk.  Past the last chunk the operand is
    // empty and the request reads nothing.
    const auto load_w = [&](int q, int c) {
        const bool there = c < chunks;
        bring(buffer(wb, there ? n_rows * w_pitch : 0), vw[q], (c & 1) * G::kPart + (wave + 4 * q) * 1024, there ? (c - first) * 128 : 0);
    };
    const auto load_x = [&](int q, int t) {          // t: chunk, or half chunk
        const int halves = kFour ? 1 : 2;
        const bool there = t < halves * chunks;
        bring(buffer(xb, there ? m_rows * x_pitch : 0), vx[q], G::kX + (t & 1) * G::kPart + (wave + 4 * q) * 1024,
              there ? (t - halves * first) * 128 : 0);
    };

    // Scales: 32 bytes of a row are four chunks'; the last 32 are those at the row's end, wherever they start.  Rows of whole
    // words come by load-to-LDS, 32 rows at a time; others through registers, a weight row and a row of x a thread, stored a
    // chunk later.
    u32x4 sw[2] = {}, sx[2] = {};
    const int my_w = (int)threadIdx.x < n_rows ? (int)threadIdx.x : n_rows - 1, my_x = (int)threadIdx.x < m_rows ? (int)threadIdx.x : m_rows - 1;
    const uint8_t *swp = wsb + (int64_t)my_w * blocks, *sxp = xsb + (int64_t)my_x * blocks;
    const auto start_of = [&](int u) { return 32 * u + 32 <= 8 * whole ? 32 * u : 8 * whole - 32; };
    const auto load_scales = [&](int u) {
        const int at = start_of(u);
        __builtin_memcpy(sw, swp + at, 32);
        __builtin_memcpy(sx, sxp + at, 32);
    };
    const auto bring_scales = [&](int u, int slot) {
#pragma unroll
        for (int q = 0; q < (S + 127) / 128; ++q) {
            const int r = 32 * (wave + 4 * q) + (lane >> 1), to = G::kScales + slot * G::kSlot + (wave + 4 * q) * 1024;
            bring(buffer(wsb, n_rows * blocks), (r < n_rows ? r : n_rows - 1) * blocks + (lane & 1) * 16, to, start_of(u));
            bring(buffer(xsb, m_rows * blocks), (r < m_rows ? r : m_rows - 1) * blocks + (lane & 1) * 16, to + TW * 32, start_of(u));
        }
    };
    const auto store_scales = [&](int slot) {
        u32x4* s = reinterpret_cast<u32x4*>(s_mem + G::kScales + slot * G::kSlot);
        if ((int)threadIdx.x < TW) s[2 * threadIdx.x] = sw[0], s[2 * threadIdx.x + 1] = sw[1];
        if ((int)threadIdx.x < TX) s[2 * (TW + threadIdx.x)] = sx[0], s[2 * (TW + threadIdx.x) + 1] = sx[1];
    };
    const auto four_bytes = [](const uint8_t* p) {
        uint32_t v;
        __builtin_memcpy(&v, p, 4);
        return v;
    };
    const auto part_bytes = [&](const uint8_t* p, int from) {          // of the blocks that are none: 2^0
        uint32_t v = 0x7F7F7F7Fu;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (from + i < part) v = (v & ~(0xFFu << (8 * i))) | (uint32_t)p[8 * whole + from + i] << (8 * i);
        return v;
    };
    // Where the scales of chunk c are, from those of the first chunk of slot 0 on.
    const auto scales_of = [&](int c) {
        const int f = c - first, u = f >> 2;
        return f < 0 ? G::kSlot : (u & 1) * G::kSlot + 8 * f - (whole < 4 ? 0 : start_of(u));
    };

    // e2m1: a lane's blocks of a chunk are 4 h .. 4 h + 3, h = lane / 32, one for each of four instructions along k, their scales a
    // word.  e4m3: of either half of a chunk a lane, g = lane / 16, has the weight's block g, and of x the pieces g and 4 + g.
    const int w_row = wm * (TW / 2) + row, x_row = wn * (TX / 2) + row;
    const int w_at = w_row * 128 + (((kFour ? 4 * part_of : part_of) ^ (row >> 1)) & 7) * 16;
    const int x_at = G::kX + x_row * 128 + (((kFour ? 4 * part_of : part_of) ^ (row >> 1)) & 7) * 16;
    const int s_at = G::kScales + (kFour ? 4 * part_of : part_of);
    const auto read = [&](int at) { return *reinterpret_cast<const u32x4*>(s_mem + at); };

    Sums acc[WT][XT];
#pragma unroll
    for (int i = 0; i < WT; ++i)
#pragma unroll
        for (int j = 0; j < XT; ++j) acc[i][j] = Sums{};
    // here, and not behind the next wait, where the compiler would put what has no use before it
    const auto pin = [](Sums& c) {
        if constexpr (S == 256) asm volatile("" : "+a"(c));
        else asm volatile("" : "+v"(c));
    };
    const auto hand_over = [] {
        __builtin_amdgcn_s_waitcnt(0x0070);          // vmcnt(0), lgkmcnt(0)
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };

    // A column's bias a thread until the end, where LDS hands it round: more would be registers that the products need, and asked for
    // there it is waited for (8192 by 4096 x 12288 in 4 bits 298 us, 264 so, and 250 without a bias).
    float my_bias = 0.f;
    if constexpr (BIAS) my_bias = T::to_f32(bias[n0 + (int)threadIdx.x % TW < N ? n0 + (int)threadIdx.x % TW : N - 1]);
    // ---- before the first chunk: requests first, what the waves bring themselves behind them ----
    if (!part) {
#pragma unroll
        for (int q = 0; q < G::kLoads; ++q) load_w(q, 0), load_x(q, 0);
        if (!kFour) {
#pragma unroll
            for (int q = 0; q < G::kLoads; ++q) load_x(q, 1);
        }
    }
    // What goes out behind the barrier of a chunk that does not exist.  (In e2m1, and in e4m3 tiles of 256, a part of it goes out
    // in the first chunk's steps once more, to the same place, which nobody reads before the barrier behind both.)
    if (kFour) {
#pragma unroll
        for (int q = 0; q < G::kLoads; ++q) load_w(q, 1), load_x(q, 1);
    } else {
#pragma unroll
        for (int q = 0; q < G::kLoads / 2; ++q) load_w(q, 1);
    }
    if (whole >= 4) {
        if (words) bring_scales(0, 0);
        else load_scales(0);
    } else {
#pragma unroll
        for (int i = 0; i < 6; ++i)
            if (i < 2 * whole) sw[i >> 2][i & 3] = four_bytes(swp + 4 * i), sx[i >> 2][i & 3] = four_bytes(sxp + 4 * i);
    }
    if (!words || whole < 4) store_scales(0);
    if (part) {
        sw[0][0] = part_bytes(swp, 0), sw[0][1] = part_bytes(swp, 4), sx[0][0] = part_bytes(sxp, 0), sx[0][1] = part_bytes(sxp, 4);
        store_scales(1);
#pragma unroll
        for (int q = 0; q < G::kLoads; ++q) {
            const int to = (wave + 4 * q) * 1024 + lane * 16;
            u32x4 v = {0, 0, 0, 0};
            if (piece < part) v = *reinterpret_cast<const u32x4*>(wb + vw[q] + whole * 128);
            *reinterpret_cast<u32x4*>(s_mem + to) = v;
#pragma unroll
            for (int h = 0; h < (kFour ? 1 : 2); ++h) {
                v = u32x4{0, 0, 0, 0};
                if (kFour ? piece < part : 8 * h + piece < 2 * part) v = *reinterpret_cast<const u32x4*>(xb + vx[q] + whole * (kFour ? 128 : 256) + h * 128);
                *reinterpret_cast<u32x4*>(s_mem + G::kX + h * G::kPart + to) = v;
            }
        }
    }
    hand_over();
    // the scales of four chunks, three to four chunks ahead; through registers those loaded a chunk ago
    const auto scales_ahead = [&](int c) {
        const int f = c - first, u = (f >> 2) + 1;
        if (f < 0 || 4 * u >= whole) return;
        if (!words && (f & 3) == 1) store_scales(u & 1);
        if ((f & 3) == 0) {
            if (words) bring_scales(u, u & 1);
            else load_scales(u);
        }
    };

    if constexpr (kFour) {
        // Four steps a chunk, an instruction along k each: WT x XT products on fragments that the step before has read.
        u32x4 a[2][WT], b[2][XT];
        uint32_t as[WT], bs[XT], an[WT], bn[XT];      // an, bn: the next chunk's
        const auto read_scales = [&](int c, uint32_t (&a4)[WT], uint32_t (&b4)[XT]) {
            const int s = s_at + scales_of(c < chunks ? c : chunks - 1);
#pragma unroll
            for (int i = 0; i < WT; ++i) a4[i] = *reinterpret_cast<const uint32_t*>(s_mem + s + (w_row + i * R) * 32);
#pragma unroll
            for (int j = 0; j < XT; ++j) b4[j] = *reinterpret_cast<const uint32_t*>(s_mem + s + (TW + x_row + j * R) * 32);
        };
        read_scales(0, as, bs);
#pragma unroll
        for (int i = 0; i < WT; ++i) a[0][i] = read(w_at + i * R * 128);
#pragma unroll
        for (int j = 0; j < XT; ++j) b[0][j] = read(x_at + j * R * 128);
        const auto step = [&](auto ks_, int c) {
            constexpr int ks = decltype(ks_)::value, p = ks & 1;
            if constexpr (ks == 3) {
                hand_over();
                read_scales(c + 1, an, bn);
            }
            const int at = ks == 3 ? ((c + 1) & 1) * G::kPart : (c & 1) * G::kPart, k16 = ks == 3 ? 0 : (ks + 1) * 16;
            constexpr int kSlots = 2 * XT;           // requests for chunk c + 2 (or those still to make for c + 1): steps 3 and 0
#pragma unroll
            for (int j = 0; j < XT; ++j) {
                // the next step's fragments
                b[1 - p][j] = read(((at + x_at) ^ k16) + j * R * 128);
                a[1 - p][j] = read(((at + w_at) ^ k16) + j * R * 128);
                if constexpr (ks == 3 || ks == 0) {
                    constexpr int s0 = ks == 3 ? 0 : XT * (ks + 1);
                    const int target = ks == 3 ? c + 2 : c + 1;
#pragma unroll
                    for (int q = (s0 + j) * 2 * G::kLoads / kSlots; q < (s0 + j + 1) * 2 * G::kLoads / kSlots; ++q)
                        q & 1 ? load_w(q / 2, target) : load_x(q / 2, target);
                }
#pragma unroll
                for (int i = 0; i < WT; ++i) {
                    acc[i][j] = mfma32<ks>(a[p][i], b[p][j], acc[i][j], as[i], bs[j]);
                    pin(acc[i][j]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
            scales_ahead(c);
            step(Const<0>(), c);
            step(Const<1>(), c);
            step(Const<2>(), c);
            step(Const<3>(), c);
#pragma unroll
            for (int i = 0; i < WT; ++i) as[i] = an[i];
#pragma unroll
            for (int j = 0; j < XT; ++j) bs[j] = bn[j];
        }
    } else {
        // Half a chunk, 128 values, is XT steps of WT products: the weight's fragments stay, those of x come two steps ahead.  The
        // last step reads each weight fragment of the next half as soon as its last product has gone out.  x has a buffer for
        // either half, asked for again half a chunk later, the weight's loads are dealt over both halves.
        struct FragmentX {
            u32x4 lo, hi;
            uint32_t scale;
        };
        u32x4 a[WT];
        uint32_t as[WT];
        FragmentX b[4];
        const auto read_w = [&](int i, int t, int s) {
            a[i] = read((((t >> 1) & 1) * G::kPart + w_at + i * R * 128) ^ ((t & 1) * 64));
            as[i] = s_mem[s + (w_row + i * R) * 32];
        };
        const auto read_x = [&](FragmentX& f, int j, int t, int s) {
            const int at = (t & 1) * G::kPart + x_at + j * R * 128;
            f.lo = read(at), f.hi = read(at ^ 64);
            f.scale = s_mem[s + (TW + x_row + j * R) * 32];
        };
        const int halves = 2 * chunks;
        const auto scales_at = [&](int t) { return s_at + scales_of(t >> 1) + (t & 1) * 4; };
        {
            const int s = scales_at(0);
#pragma unroll
            for (int i = 0; i < WT; ++i) read_w(i, 0, s);
            read_x(b[0], 0, 0, s), read_x(b[1], 1, 0, s);
        }
        constexpr int kAll = G::kLoads + G::kLoads / 2, kSpread = XT >= 8 ? 3 : 2, kStep = (kAll + kSpread - 1) / kSpread;
#pragma unroll 1
        for (int t = 0; t < halves; ++t) {
            if ((t & 1) == 0) scales_ahead(t >> 1);
            const int tn = t + 1 < halves ? t + 1 : t, s = scales_at(t), sn = scales_at(tn);
#pragma unroll
            for (int j = 0; j < XT; ++j) {
                if (j == XT - 2) hand_over();
                // behind the barrier of half t the requests for half t + 2, and half of those for a chunk of the weight
                const int slot = (j + 2) % XT, target = j >= XT - 2 ? t + 2 : t + 1;
                if (slot < kSpread) {
#pragma unroll
                    for (int q = slot * kStep; q < (slot + 1) * kStep && q < kAll; ++q) {
                        if (q < G::kLoads) {
                            load_x(q, target);
                        } else {
                            const int half = (target & 1) ? 0 : G::kLoads / 2, qw = q - G::kLoads;
                            if (half) load_w(qw + G::kLoads / 2, (target + 1) >> 1);
                            else load_w(qw, (target + 1) >> 1);
                        }
                    }
                }
                if (j + 2 < XT) read_x(b[(j + 2) & 3], j + 2, t, s);
                else read_x(b[(j + 2) & 3], j + 2 - XT, tn, sn);
#pragma unroll
                for (int i = 0; i < WT; ++i) {
                    acc[i][j] = mfma<FORMAT>(a[i], b[j & 3].lo, b[j & 3].hi, acc[i][j], as[i], b[j & 3].scale);
                    pin(acc[i][j]);
                    if (j == XT - 1) {
                        __builtin_amdgcn_sched_barrier(0);
                        read_w(i, tn, sn);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    // ---- the tile, row by row: R rows of x and TW / 2 weight rows at a time through LDS, a wave on its own ----
    using E = typename T::elem;
    constexpr int kQ = R * R / 256, kV = 16 / sizeof(E), kPitch = TW / 2 * sizeof(E) + 16;
    static_assert(4 * R * kPitch + TW * 4 <= G::kLds, "");
    const int64_t n_wave = n0 + wm * (TW / 2), m_wave = m0 + wn * (TX / 2);
    const bool full = n_wave + TW / 2 <= N;      // and else a row ends in the tile
    float* s_bias = reinterpret_cast<float*>(s_mem + 4 * R * kPitch);
    const auto value = [&](int i, int j, int q) {
        f32x4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        if constexpr (BIAS) v += *reinterpret_cast<const f32x4*>(s_bias + wm * (TW / 2) + i * R + 8 * q + 4 * part_of);
        return v;
    };
    hand_over();             // nobody reads a chunk any more, and no request, the empty ones among them, is on its way to LDS
    if constexpr (BIAS) {
        if ((int)threadIdx.x < TW) s_bias[threadIdx.x] = my_bias;
        __syncthreads();
    }
    unsigned char* s_out = s_mem + wave * R * kPitch;
#pragma unroll
    for (int j = 0; j < XT; ++j) {
#pragma unroll
        for (int i = 0; i < WT; ++i)
#pragma unroll
            for (int q = 0; q < kQ; ++q) {
                const f32x4 v = value(i, j, q);
                unsigned char* to = s_out + row * kPitch + (i * R + 8 * q + 4 * part_of) * sizeof(E);
                if constexpr (sizeof(E) == 4) *reinterpret_cast<f32x4*>(to) = v;
                else *reinterpret_cast<u32x2*>(to) = u32x2{T::pack2(v[0], v[1]), T::pack2(v[2], v[3])};
            }
        __builtin_amdgcn_wave_barrier();
        constexpr int kLanes = TW / 2 / kV;      // of a row
#pragma unroll
        for (int q = 0; q < R * kLanes / 64; ++q) {
            const int r = (q * 64 + lane) / kLanes, c = (q * 64 + lane) % kLanes;
            const unsigned char* from = s_out + r * kPitch + c * 16;
            const int64_t m = m_wave + j * R + r, n = n_wave + c * kV;
            const u32x4 v = *reinterpret_cast<const u32x4*>(from);
            if (m >= rows) continue;
            if (full) {
                __builtin_memcpy(y + m * N + n, &v, 16);     // any address of the type
            } else {
#pragma unroll 1
                for (int e = 0; e < kV; ++e)
                    if (n + e < N) y[m * N + n + e] = reinterpret_cast<const E*>(from)[e];
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <typename T, int FORMAT, int S, bool BIAS>
hipError_t launch(const Product& p, hipStream_t stream) {
    using G = Tiles<FORMAT, S>;
    using E = typename T::elem;
    const int x_tiles = (int)cdiv(p.rows, S), w_tiles = (int)cdiv(p.n, S);
    if (const hipError_t e = allow_lds<&mx_tiles_kernel<T, FORMAT, S, BIAS>>(G::kLds); e != hipSuccess) return e;
    const unsigned grid = (unsigned)(cdiv((int64_t)x_tiles * w_tiles, 8) * 8);
    const int words = p.k / kBlock % 4 == 0 && ((reinterpret_cast<uintptr_t>(p.ws) | reinterpret_cast<uintptr_t>(p.xs)) & 3) == 0;
    return start(&mx_tiles_kernel<T, FORMAT, S, BIAS>, dim3(grid), G::kThreads, G::kLds, stream, p.x, p.xs, p.w, p.ws,
                 static_cast<const E*>(p.bias), static_cast<E*>(p.y), (int)p.rows, (int)p.n, (int)(p.k / kBlock), words, x_tiles, w_tiles);
}

}  // namespace

int tiles_product(const Product& p, int tile, hipStream_t stream) {
    hipError_t e = hipSuccess;
    by_type(p.dtype, p.format, [&](auto t, auto f) {
        using T = decltype(t);
        constexpr int F = decltype(f)::value;
        if (p.bias) e = tile == 256 ? launch<T, F, 256, true>(p, stream) : launch<T, F, 128, true>(p, stream);
        else e = tile == 256 ? launch<T, F, 256, false>(p, stream) : launch<T, F, 128, false>(p, stream);
    });
    return hip_status("mx_tiles_kernel", e);
}

}  // namespace nqx
