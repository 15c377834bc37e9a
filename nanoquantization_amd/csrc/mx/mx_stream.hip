// The product for a few rows of x, or few tiles of 128, where what counts is to stream the packed weight once: 0.53 bytes a value,
// and all of x per workgroup.  A workgroup has 128 weight rows, up to 128 rows of x and a run of k.  Operands come to LDS by
// load-to-LDS in chunks of 256 values of k, whole 128-byte lines of a weight row, two chunks ahead of the one that is multiplied;
// one barrier a chunk.  (x comes from a cache, but its requests return behind the weight's: asked for one chunk ahead a chunk of 64
// rows took 2.5 us.  Three chunks ahead gain nothing: 41 rows by 25600 x 5120 in 4 bits 21.6 us and 21.4.)  Where the weight has too
// few rows for the chip, k is split over workgroups, whose sums go to memory in fp32 and are added, in the order of the splits, by a
// second kernel.  Up to 64 rows are bound by the weight's bytes (16 by 5120 x 25600 12.5 us, 5.6 TB/s, with the weight in the last cache,
// and 16.6 from memory).  More rows: a wave reads a chunk's fragments behind its barrier and then multiplies them, and with all waves in
// step the two hardly overlap (333 by 2816 x 9728 in 8 bits 1.1 us a chunk: 0.5 us of matrix instructions, and 0.7 without them).
//
// With RAW x comes as it is and every workgroup quantises its run of it into LDS first, while its first chunks are on their way:
// one launch for a linear of few rows.
#include "mx_linear.hpp"

namespace nqx {
namespace {

constexpr int kRows = 128;      // weight rows of a workgroup
// By sixteens of rows of x: chunks whose scales come at a time, workgroups that fit a CU's LDS, and how many fours of waves a
// workgroup has: of two, one has a chunk's first instruction along k and one the second, so that a SIMD has something else to do
// while a wave waits for LDS.
constexpr int group_chunks(int mt) { return mt >= 4 ? 2 : 4; }
constexpr int per_cu(int mt) { return mt == 1 ? 2 : 1; }
constexpr int fours(int mt) { return mt == 1 ? 1 : 2; }
int chunks_of(int64_t k) { return (int)cdiv(k, 256); }
int sixteens(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : rows <= 64 ? 4 : 8; }
// Splits of k: at most as many as fill the chip with workgroups that are resident at once, of four chunks each at least, and of those
// the number that costs least: the longest split's chunks or, if that is more, the weight's way from memory, and where there is more
// than one a launch and the sums' way to memory and back.  Nanoseconds of a chunk and of a launch and 5.2 TB/s as measured; 128 rows by 2560 x 9728 in 8 bits 18.0 us with two splits and 15.2
// with one, 64 rows in 4 bits 11.7 and 9.5; 16 rows by 5120 x 25600, from
// memory, 20.2 and 16.7.  (Workgroups of 256 weight rows would share x among more of them: 41 rows by
// 25600 x 5120 26.5 us and 24.5 with 128, 64 rows by 4096 x 12288 17.6 and 14.3.)
int splits_of(int64_t rows, int64_t n, int64_t k, int format) {
    const int mt = sixteens(rows);
    const int64_t tiles = cdiv(n, kRows) * cdiv(rows, 16 * mt), chunks = chunks_of(k), chunk = mt == 8 ? (format == NQX_FP4 ? 730 : 1070) : mt == 1 ? 600 : 700;
    int64_t most = 256 * per_cu(mt) / tiles;
    if (most > k / 1024) most = k / 1024;
    if (most > 16) most = 16;
    const int64_t least = n * (k * 17 / 32) / 5200;          // the weight's way from memory
    int64_t best = 1, time = 0;
    for (int64_t s = 1; s <= most || s == 1; ++s) {
        int64_t t = cdiv(chunks, s) * chunk;
        if (t < least) t = least;
        if (s > 1) t += 3000 + s * rows * n * 8 / 5200;
        if (s == 1 || t < time) best = s, time = t;
    }
    return (int)best;
}
template <int FORMAT, int MT, bool RAW>
struct Stream {
    static constexpr int kFours = fours(MT), kWaves = 4 * kFours, kThreads = 64 * kWaves, kBufs = 3;
    static constexpr int kGroup = group_chunks(MT), kBytes = 8 * kGroup;       // chunks whose scales come at a time, a row's bytes of them
    // fragments of a wave: four waves along the weight rows, or two along them and two along 128 rows of x
    static constexpr int kAlong = MT == 8 ? 2 : 1, kWT = kRows / 64 * kAlong, kXT = MT / kAlong;
    static constexpr int kHalves = FORMAT == NQX_FP4 ? 1 : 2;          // 128-byte parts of a row of x in a chunk
    static constexpr int kW = kRows * 128, kXHalf = 16 * MT * 128, kX = RAW ? 0 : kHalves * kXHalf, kXAt = kBufs * kW;      // [weight | x]
    // load-to-LDS of a wave for a chunk, 1 KiB each
    static constexpr int kWLoads = kRows / 8 / kWaves, kXAll = RAW ? 0 : 2 * MT * kHalves, kXLoads = (kXAll + kWaves - 1) / kWaves;
    static constexpr int kLoads = kWLoads + kXLoads;
    static constexpr int kNone = kXAt + kBufs * kX;                         // where a wave without a piece of x lets its request go
    static constexpr int kScales = kNone + (kXAll % kWaves ? 1024 : 0), kSlot = (kRows + (RAW ? 0 : 16 * MT)) * kBytes;
    static constexpr int kFixed = kScales + 2 * kSlot;
    static constexpr int kSumPitch = kRows + 4;      // floats of a row of sums of two fours, in the buffers' place
    static_assert(kFours == 1 || 16 * MT * kSumPitch * 4 <= kNone, "");
    static_assert(kFixed * per_cu(MT) <= 160 * 1024, "");
};
// RAW: bytes of `rows` quantised rows of `chunks` chunks in LDS, codes and scales.
__host__ __device__ constexpr int resident_bytes(int format, int rows, int chunks) {
    return rows * chunks * ((format == NQX_FP4 ? 128 : 256) + 8);
}

template <typename T, int FORMAT, int MT, bool RAW>
__global__ __launch_bounds__(256 * fours(MT)) void mx_stream_kernel(const void* __restrict__ x, int64_t x_stride, const uint8_t* __restrict__ xs,
                                                        const uint8_t* __restrict__ w, const uint8_t* __restrict__ ws,
                                                        const typename T::elem* __restrict__ bias, typename T::elem* __restrict__ y,
                                                        float* __restrict__ sums, int rows, int N, int blocks, int words, int each, int more,
                                                        uint32_t row_tiles) {
    using G = Stream<FORMAT, MT, RAW>;
    constexpr bool kFour = FORMAT == NQX_FP4;
    constexpr int kWaves = G::kWaves, kThreads = G::kThreads, kWT = G::kWT, kXT = G::kXT, kGroup = G::kGroup, kBytes = G::kBytes;
    extern __shared__ __attribute__((aligned(16))) unsigned char s_mem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lo = lane & 15, hi = lane >> 4;
    // The row tiles of a weight tile run next to each other on one XCD (workgroups go round the eight of them), whose L2 then has
    // the weight for all but the first: 333 rows by 2816 x 9728 in 8 bits 17.8 us, 18.1 across XCDs; 1000 by 4096 x 4096 24.5 and 26.5.
    // row_tiles is 1 where they lie along blockIdx.z: one tile, or an XCD would have more workgroups than CUs.
    const uint32_t turn = blockIdx.x >> 3, tile = row_tiles == 1 ? blockIdx.x : turn / row_tiles * 8 + (blockIdx.x & 7);
    const int split = blockIdx.y, n0 = (int)(tile * kRows), m0 = (int)(row_tiles == 1 ? blockIdx.z : turn % row_tiles) * (16 * MT);
    if (n0 >= N) return;
    const int n_rows = N - n0 < kRows ? N - n0 : kRows, all_rows = rows;
    rows = rows - m0 < 16 * MT ? rows - m0 : 16 * MT;
    const uint32_t w_pitch = (uint32_t)blocks * 16, x_pitch = (uint32_t)blocks * (kFour ? 16 : 32);
    // Chunks: the blocks that do not fill one come first (pieces that do not exist are asked for past the buffer's end, which
    // leaves zeros), then the whole ones.  A split has a run of them, the first `more` splits one more than the others.  Scales come for
    // a group of chunks at a time, kBytes of a row: for the chunk that is not whole, then for kGroup whole ones each.
    const int part = blocks & 7, whole = blocks >> 3, first = part ? 1 : 0;
    const int c0 = split * each + min(split, more), c1 = c0 + each + (split < more ? 1 : 0);
    const auto group_of = [&](int c) { return c < first ? 0 : first + (c - first) / kGroup; };
    const auto chunk_of = [&](int g) { return g < first ? 0 : first + kGroup * (g - first); };       // a group's first
    const int g0 = group_of(c0), g1 = group_of(c1 - 1) + 1;

    const uint8_t *wb = w + (int64_t)n0 * w_pitch, *wsb = ws + (int64_t)n0 * blocks, *xb = static_cast<const uint8_t*>(x) + (RAW ? 0 : (int64_t)m0 * x_pitch);
    if constexpr (!RAW) xs += (int64_t)m0 * blocks;
    const auto buffer = [](const uint8_t* p, uint32_t bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, bytes, 0x00020000);
    };
    const auto bring = [&](__amdgpu_buffer_rsrc_t r, uint32_t v, int to, int from) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(s_mem + to), 16, v, from, 0, 0);
    };
    // A load-to-LDS writes 1 KiB in the order of the lanes: eight rows of 128 bytes.  A row's 16-byte pieces are stored at position
    // piece ^ (row / 2 % 8), which spreads the 16 rows of a fragment read over all banks; the swizzle is in the source addresses.
    // Rows past an operand's end are past its buffer's: zeros.
    constexpr uint32_t kNowhere = 0x7FFFFFF0u;       // past the end of every buffer
    const auto swizzle = [](int row, int piece) { return (piece ^ (row >> 1)) & 7; };
    uint32_t vw[G::kWLoads], vx[G::kXLoads ? G::kXLoads : 1];
    int x_half[G::kXLoads ? G::kXLoads : 1], x_to[G::kXLoads ? G::kXLoads : 1];       // of a wave's loads of x: half, place
    bool x_mine[G::kXLoads ? G::kXLoads : 1];
    const int piece = swizzle(8 * wave + (lane >> 3), lane & 7);            // of all a lane's loads: their rows are 32 apart
#pragma unroll
    for (int q = 0; q < G::kWLoads; ++q) vw[q] = (8 * (wave + kWaves * q) + (lane >> 3)) * w_pitch + piece * 16;
#pragma unroll
    for (int q = 0; q < G::kXLoads; ++q) {
        const int i = wave + kWaves * q, r = 8 * (i % (2 * MT)) + (lane >> 3);
        x_mine[q] = i < G::kXAll, x_half[q] = i / (2 * MT), x_to[q] = i * 1024;
        vx[q] = x_mine[q] ? r * x_pitch + swizzle(r, lane & 7) * 16 + x_half[q] * 128 : kNowhere;
    }
    // Chunk c, or nothing past the last, to buffer `ring`.  PARTIAL: it may be the one that is not whole.
    const auto load = [&](auto partial_, int c, int ring) {
        constexpr bool PARTIAL = decltype(partial_)::value != 0;
        const bool there = c < c1, partial = PARTIAL && c < first;
        const int f = there ? partial ? whole : c - first : 0;
        const auto bw = buffer(wb, there ? n_rows * w_pitch : 0), bx = buffer(xb, there ? rows * x_pitch : 0);
#pragma unroll
        for (int q = 0; q < G::kWLoads; ++q)
            bring(bw, PARTIAL && partial && piece >= part ? kNowhere : vw[q], ring * G::kW + (wave + kWaves * q) * 1024, f * 128);
#pragma unroll
        for (int q = 0; q < G::kXLoads; ++q) {
            const int r = 8 * ((wave + kWaves * q) % (2 * MT)) + (lane >> 3), p = swizzle(r, lane & 7);
            const bool none = PARTIAL && partial && (kFour ? p >= part : 8 * x_half[q] + p >= 2 * part);
            bring(bx, none ? kNowhere : vx[q], x_mine[q] ? G::kXAt + ring * G::kX + x_to[q] : G::kNone, f * 128 * G::kHalves);
        }
    };
    const auto start_of = [&](int g) {               // where the bytes begin: kBytes of the row are left at most
        const int at = g < first ? 8 * whole : kBytes * (g - first), last = (g < first ? blocks : 8 * whole) - kBytes;
        return at < last ? at : last < 0 ? 0 : last;
    };
    constexpr int kScaleRows = G::kSlot / kBytes, kLanes = kBytes / 16;        // lanes of a row in a load-to-LDS
    constexpr int kTurns = (kScaleRows + kThreads - 1) / kThreads;
    u32x4 sv[kTurns][kLanes] = {};
    // Rows of whole words come by load-to-LDS; others, and short ones, through registers, a row a thread or two.
    const auto ask_scales = [&](int g) {
        if (g >= g1) return;
        const int at = start_of(g), slot = G::kScales + (g & 1) * G::kSlot;
        if (words) {
#pragma unroll
            for (int i = 0; i < (kRows * kLanes + kThreads - 1) / kThreads; ++i) {
                const int e = kThreads * i + threadIdx.x;
                if (kRows * kLanes % kThreads == 0 || kThreads * i + 64 * wave < kRows * kLanes)
                    bring(buffer(wsb, n_rows * blocks), e / kLanes * blocks + e % kLanes * 16, slot + (kWaves * i + wave) * 1024, at);
            }
            if constexpr (!RAW) {
                // 16 rows of x are less than a request's: the other lanes' are past the slot
#pragma unroll
                for (int i = 0; i < (16 * MT * kLanes + kThreads - 1) / kThreads; ++i) {
                    const int e = kThreads * i + threadIdx.x;
                    if (e < 16 * MT * kLanes)
                        bring(buffer(xs, rows * blocks), e / kLanes * blocks + e % kLanes * 16, slot + kRows * kBytes + (kWaves * i + wave) * 1024, at);
                }
            }
        } else {
#pragma unroll
            for (int t = 0; t < kTurns; ++t) {
                const int r = threadIdx.x + t * kThreads;
                if (r >= kScaleRows) break;
                const uint8_t* from = r < kRows ? wsb + (int64_t)(r < n_rows ? r : n_rows - 1) * blocks
                                                : xs + (int64_t)(r - kRows < rows ? r - kRows : rows - 1) * blocks;
                if (blocks >= kBytes) {
                    __builtin_memcpy(sv[t], from + at, kBytes);
                    continue;
                }
#pragma unroll
                for (int i = 0; i < kBytes / 4; ++i) {
                    uint32_t v = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (4 * i + e < blocks) v |= (uint32_t)from[4 * i + e] << (8 * e);
                    sv[t][i / 4][i % 4] = v;
                }
            }
        }
    };
    const auto put_scales = [&](int g) {
        if (words || g >= g1) return;
#pragma unroll
        for (int t = 0; t < kTurns; ++t) {
            const int r = threadIdx.x + t * kThreads;
            if (r >= kScaleRows) break;
            u32x4* s = reinterpret_cast<u32x4*>(s_mem + G::kScales + (g & 1) * G::kSlot) + kLanes * r;
#pragma unroll
            for (int i = 0; i < kLanes; ++i) s[i] = sv[t][i];
        }
    };

    f32x4 acc[kWT][kXT];
#pragma unroll
    for (int i = 0; i < kWT; ++i)
#pragma unroll
        for (int j = 0; j < kXT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // Columns and bias of a lane at the end: with two fours those of its 16 bytes of a row, else four for each of its fragments.
    constexpr int V = G::kFours == 2 ? 16 / sizeof(typename T::elem) : 4, kOf = kRows / V;
    const int column = G::kFours == 2 ? threadIdx.x % kOf * V : wave * (16 * kWT) + 4 * hi;
    float b[G::kFours == 2 ? 1 : kWT][V] = {};
    if (bias && gridDim.y == 1) {
#pragma unroll
        for (int i = 0; i < (G::kFours == 2 ? 1 : kWT); ++i) load_bias<T>(b[i], bias, n0 + column + 16 * i, N);
    }
    ask_scales(g0);
    load(Const<1>(), c0, 0);
    load(Const<0>(), c0 + 1, 1);
    const int chunks = c1 - c0, r_bytes = chunks * (kFour ? 128 : 256);      // RAW: of a row's codes in LDS; the scales behind all of them
    unsigned char* s_x = s_mem + G::kFixed;
    unsigned char* s_xs = s_x + rows * r_bytes;
    if constexpr (RAW) {
        // rows x the run of k: a lane eight values, four lanes a block; what is not there becomes zeros
        using E = typename T::elem;
        const int per_row = chunks * 32;
        for (int r = 0; r < rows; ++r)
            for (int e = threadIdx.x; e < per_row; e += kThreads) {
                const int c = c0 + (e >> 5), in_chunk = (e & 31) * 8, at = 256 * (c < first ? whole : c - first) + in_chunk;
                Eight<T, FORMAT> v;
                v.clear();
                if (at < blocks * 32) v.load(static_cast<const E*>(x) + r * x_stride + at);
                uint32_t byte;
                const u32x2 code = v.encode(byte);
                const int b = in_chunk >> 5, within = in_chunk & 31;               // block of the chunk
                if constexpr (kFour) {
                    *reinterpret_cast<uint32_t*>(s_x + r * r_bytes + (c - c0) * 128 + swizzle(r, b) * 16 + within / 2) = code.x;
                } else {
                    const int h = b >> 2, p = (b & 3) * 2 + (within >> 4);
                    *reinterpret_cast<u32x2*>(s_x + r * r_bytes + (c - c0) * 256 + h * 128 + swizzle(r, p) * 16 + (within & 15)) = code;
                }
                if ((e & 3) == 0) s_xs[r * chunks * 8 + (c - c0) * 8 + b] = (unsigned char)byte;
            }
    }
    put_scales(g0);

    // The chunk's eight blocks in two instructions: lane group g has the blocks 2 g and 2 g + 1, whose scales are next to each other.
    // Where a lane's pieces are for the first, from a fragment's first row on; for the second they are a piece (e2m1, and the
    // weight) or two (e4m3) on, before the swizzle.
    const int own = wave & 3, mine = wave >> 2;      // quarter of the weight rows; of two fours the instruction along k
    const int wm = own % (4 / G::kAlong), wn = own / (4 / G::kAlong);
    const int w_row = wm * (16 * kWT) + lo, x_row = wn * (16 * kXT) + lo, x_own = lo < rows ? lo : rows - 1;
    const int w_at = w_row * 128 + swizzle(lo, 2 * hi) * 16;
    const int x_piece = kFour ? 2 * hi : 4 * (hi >> 1) + (hi & 1);
    const int x_at = RAW ? G::kFixed + x_own * r_bytes + swizzle(x_own, x_piece) * 16 : G::kXAt + x_row * 128 + swizzle(lo, x_piece) * 16;
    const auto read = [&](int at) { return *reinterpret_cast<const u32x4*>(s_mem + at); };
    int ring = 0, g = g0, s_at = 0, left = 0;
    const auto chunk = [&](auto partial_, int c) {
        constexpr bool PARTIAL = decltype(partial_)::value != 0;
        // chunk c has landed, c + 1 may be on its way; nobody needs the buffers of c - 1 any more
        __builtin_amdgcn_s_waitcnt(0x0070 | (G::kLoads & 15) | (G::kLoads >> 4) << 14);       // vmcnt(kLoads), lgkmcnt(0)
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        const bool begins = left == 0;
        if (begins) {
            // where the group's first chunk has its scales, and how many chunks it has
            s_at = G::kScales + (g & 1) * G::kSlot + 8 * (PARTIAL ? whole : c - first) - start_of(g);
            left = chunk_of(g + 1) - c;
            ask_scales(g + 1);
        }
        load(Const<0>(), c + 2, ring == 0 ? 2 : ring - 1);
        // of the chunk that is not whole a block that is none has zeros for codes and the scale of the last block, which is no NaN unless
        // the row's sum is
        const auto scales = [&](int at) -> uint32_t {
            if constexpr (PARTIAL) {
                const int b0 = min(2 * hi, part - 1), b1 = min(2 * hi + 1, part - 1);
                return s_mem[at + b0] | (uint32_t)s_mem[at + b1] << 8;
            } else {
                return *reinterpret_cast<const uint16_t*>(s_mem + at + 2 * hi);
            }
        };
        uint32_t as[kWT], bs[kXT];
#pragma unroll
        for (int i = 0; i < kWT; ++i) as[i] = scales(s_at + (w_row + 16 * i) * kBytes);
#pragma unroll
        for (int j = 0; j < kXT; ++j) {
            if constexpr (RAW) bs[j] = *reinterpret_cast<const uint16_t*>(s_xs + x_own * chunks * 8 + (c - c0) * 8 + 2 * hi);
            else bs[j] = scales(s_at + (kRows + x_row + 16 * j) * kBytes);
        }
        const int wp = ring * G::kW + w_at, xp = x_at + (RAW ? (c - c0) * (kFour ? 128 : 256) : ring * G::kX);
        const auto half = [&](auto h_) {
            constexpr int h = decltype(h_)::value;
            u32x4 a[kWT];
#pragma unroll
            for (int i = 0; i < kWT; ++i) a[i] = read((wp ^ (16 * h)) + i * 2048);
#pragma unroll
            for (int j = 0; j < kXT; ++j) {
                u32x4 x0, x1;
                if constexpr (kFour) {
                    x0 = x1 = read((xp ^ (16 * h)) + j * 2048);
                } else {
                    x0 = read((xp ^ (32 * h)) + j * 2048);
                    x1 = read((xp ^ (32 * h)) + j * 2048 + (RAW ? 128 : G::kXHalf));
                }
#pragma unroll
                for (int i = 0; i < kWT; ++i) acc[i][j] = mfma<FORMAT, h>(a[i], x0, x1, acc[i][j], as[i], bs[j]);
            }
        };
        if constexpr (G::kFours == 1) half(Const<0>()), half(Const<1>());
        else if (mine == 0) half(Const<0>());
        else half(Const<1>());
        if (begins) put_scales(g + 1);
        s_at += 8, ring = ring == 2 ? 0 : ring + 1;
        if (--left == 0) ++g;
    };
    int c = c0;
    if (c < first) chunk(Const<1>(), c++);
#pragma unroll 1
    for (; c < c1; ++c) chunk(Const<0>(), c);
    __builtin_amdgcn_s_waitcnt(0x0F70);              // vmcnt(0): no request is on its way to LDS that is another workgroup's by then
    const int64_t pitch = ((int64_t)N + kRows - 1) / kRows * kRows;          // of a row of sums
    if constexpr (G::kFours == 2) {
        // The two fours' sums meet in LDS, and leave it row by row, 16 bytes a lane.  (Straight from the registers of one four a
        // store has 32 bytes of each of 16 rows: 333 rows by 2816 x 9727 took 20.7 us, and 18.1 so; with a bias, asked
        // for at the start, 20.0.)
        float* s_sum = reinterpret_cast<float*>(s_mem);
        const auto at = [&](int i, int j) {
            return reinterpret_cast<f32x4*>(s_sum + (x_row + 16 * j) * G::kSumPitch + wm * (16 * kWT) + 16 * i + 4 * hi);
        };
        __syncthreads();
        if (mine == 1) {
#pragma unroll
            for (int j = 0; j < kXT; ++j)
#pragma unroll
                for (int i = 0; i < kWT; ++i) *at(i, j) = acc[i][j];
        }
        __syncthreads();
        if (mine == 0) {
#pragma unroll
            for (int j = 0; j < kXT; ++j)
#pragma unroll
                for (int i = 0; i < kWT; ++i) *at(i, j) += acc[i][j];
        }
        __syncthreads();
        if (gridDim.y > 1) {
            for (int e = threadIdx.x; e < rows * (kRows / 4); e += kThreads) {
                const int r = e / (kRows / 4), c = e % (kRows / 4) * 4;
                *reinterpret_cast<f32x4*>(sums + ((int64_t)split * all_rows + m0 + r) * pitch + n0 + c) =
                    *reinterpret_cast<const f32x4*>(s_sum + r * G::kSumPitch + c);
            }
        } else if (n0 + column < N) {
            for (int r = threadIdx.x / kOf; r < rows; r += kThreads / kOf) {
                f32x4 v[V / 4];
#pragma unroll
                for (int q = 0; q < V / 4; ++q) {
                    v[q] = *reinterpret_cast<const f32x4*>(s_sum + r * G::kSumPitch + column + 4 * q);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[q][i] += b[0][4 * q + i];
                }
                store_sums<T>(v, y, m0 + r, n0 + column, N);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < kWT; ++i) {
            const int n = n0 + column + 16 * i;
            if (lo >= rows || n >= N) continue;
            f32x4 v[1] = {acc[i][0]};
            if (gridDim.y > 1) {
                *reinterpret_cast<f32x4*>(sums + ((int64_t)split * all_rows + lo) * pitch + n) = v[0];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[0][e] += b[i][e];
                store_sums<T>(v, y, lo, n, N);
            }
        }
    }
}

// y = the splits' sums, added in order, + bias.
template <typename T>
__global__ __launch_bounds__(256) void mx_add_splits_kernel(const float* __restrict__ sums, const typename T::elem* __restrict__ bias,
                                                            typename T::elem* __restrict__ y, int rows, int N, int pitch, int splits) {
    // a split product has at most 256 tiles of 16 x 128 sums or 128 of up to 128 x 128: 32 bits
    const uint32_t at = (blockIdx.x * 256 + threadIdx.x) * 4, m = at / (uint32_t)pitch, n = at - m * pitch;
    if (m >= (uint32_t)rows || n >= (uint32_t)N) return;
    float b[4] = {};
    if (bias) load_bias<T>(b, bias, n, N);
    f32x4 v = *reinterpret_cast<const f32x4*>(sums + at);
    for (int s = 1; s < splits; s += 8) {            // eight on their way at once
        f32x4 next[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            next[u] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (s + u < splits) next[u] = *reinterpret_cast<const f32x4*>(sums + (int64_t)(s + u) * rows * pitch + at);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (s + u < splits) v += next[u];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += b[i];
    const f32x4 one[1] = {v};
    store_sums<T>(one, y, m, n, N);
}

template <typename T, int FORMAT, int MT, bool RAW>
hipError_t launch(const Product& p, hipStream_t stream) {
    using G = Stream<FORMAT, MT, RAW>;
    using E = typename T::elem;
    const int blocks = (int)(p.k / kBlock), tiles = (int)cdiv(p.n, kRows), splits = splits_of(p.rows, p.n, p.k, FORMAT);
    const int chunks = chunks_of(p.k);
    const int lds = G::kFixed + (RAW ? resident_bytes(FORMAT, (int)p.rows, (int)cdiv(chunks, splits)) : 0);
    if (lds > 64 * 1024)
        if (const hipError_t e = allow_lds<&mx_stream_kernel<T, FORMAT, MT, RAW>>(160 * 1024); e != hipSuccess) return e;
    const int words = blocks % 4 == 0 && blocks >= G::kBytes && ((reinterpret_cast<uintptr_t>(p.ws) | reinterpret_cast<uintptr_t>(p.xs)) & 3) == 0;
    const E *bias = static_cast<const E*>(p.bias);
    E* y = static_cast<E*>(p.y);
    const unsigned all = (unsigned)cdiv(p.rows, 16 * MT), row_tiles = cdiv(tiles, 8) * all * splits <= 32 ? all : 1;
    const dim3 grid(row_tiles == 1 ? tiles : cdiv(tiles, 8) * 8 * row_tiles, splits, row_tiles == 1 ? all : 1);
    const hipError_t e = start(&mx_stream_kernel<T, FORMAT, MT, RAW>, grid, G::kThreads, lds, stream, RAW ? p.raw : p.x, p.raw_stride, p.xs,
                               p.w, p.ws, bias, y, p.sums, (int)p.rows, (int)p.n, blocks, words, chunks / splits, chunks % splits, row_tiles);
    if (e != hipSuccess || splits == 1) return e;
    const int pitch = tiles * kRows;
    return start(&mx_add_splits_kernel<T>, dim3((unsigned)cdiv(p.rows * pitch, 1024)), 256, 0, stream, p.sums, bias, y, (int)p.rows, (int)p.n,
                 pitch, splits);
}

}  // namespace

int stream_product(const Product& p, hipStream_t stream) {
    hipError_t e = hipSuccess;
    by_type(p.dtype, p.format, [&](auto t, auto f) {
        using T = decltype(t);
        constexpr int F = decltype(f)::value;
        const int mt = sixteens(p.rows);
        if (p.raw) e = launch<T, F, 1, true>(p, stream);
        else if (mt == 1) e = launch<T, F, 1, false>(p, stream);
        else if (mt == 2) e = launch<T, F, 2, false>(p, stream);
        else if (mt == 4) e = launch<T, F, 4, false>(p, stream);
        else e = launch<T, F, 8, false>(p, stream);
    });
    return hip_status("mx_stream_kernel", e);
}

bool stream_splits(int64_t rows, int64_t n, int64_t k, int format) { return splits_of(rows, n, k, format) > 1; }
size_t stream_sums_bytes(int64_t rows, int64_t n, int64_t k, int format) {
    const int64_t splits = splits_of(rows, n, k, format);
    return splits > 1 ? (size_t)(splits * rows * cdiv(n, kRows) * kRows * 4) : 0;
}
int stream_raw_bytes(int64_t rows, int64_t n, int64_t k, int format) {
    return resident_bytes(format, (int)rows, (int)cdiv(chunks_of(k), splits_of(rows, n, k, format)));
}

}  // namespace nqx
