// The product for up to 128 rows of x, where what counts is to stream the packed weight once: 0.53 bytes a value, and all of x
// per workgroup.  A workgroup has 128 weight rows, or 256 where there is more of x to share, all rows of x and a run of k; a wave
// takes 32 weight rows.  Operands come to LDS by load-to-LDS in chunks of 256 values of k, whole 128-byte lines of a weight row,
// two chunks ahead of the one that is multiplied, or one; one barrier a chunk.  Where the weight has too few rows for the chip, k is split over workgroups, whose
// sums go to memory in fp32 and are added, in the order of the splits, by a second kernel.
//
// With RAW x comes as it is and every workgroup quantises its run of it into LDS first, while its first chunks are on their way:
// one launch for a linear of few rows.
#include "mx_linear.hpp"

namespace nqx {
namespace {

// By sixteens of rows of x: weight rows of a workgroup, buffers, and the workgroups that fit a CU's LDS.  64 rows by 5120 x 25600 with
// 128 weight rows and three buffers for any x: 26 us, 128 rows 43.
constexpr int weight_rows(int mt) { return mt >= 4 ? 256 : 128; }
constexpr int buffers(int mt) { return mt == 1 ? 3 : 2; }
constexpr int per_cu(int mt) { return mt <= 2 ? 2 : 1; }
int sixteens(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : rows <= 64 ? 4 : 8; }

template <int FORMAT, int MT, bool RAW>
struct Stream {
    static constexpr int kRows = weight_rows(MT), kWaves = kRows / 32, kThreads = 64 * kWaves, kBufs = buffers(MT);
    static constexpr int kHalves = FORMAT == NQX_FP4 ? 1 : 2;          // 128-byte parts of a row of x in a chunk
    static constexpr int kW = kRows * 128, kXHalf = 16 * MT * 128, kX = RAW ? 0 : kHalves * kXHalf, kBuf = kW + kX;
    static constexpr int kWLoads = 4, kXAll = RAW ? 0 : 2 * MT * kHalves, kXLoads = (kXAll + kWaves - 1) / kWaves;    // of a wave, 1 KiB each
    static constexpr int kLoads = kWLoads + kXLoads;
    static constexpr int kNone = kBufs * kBuf;                         // where a wave without a piece of x lets its request go
    static constexpr int kScales = kNone + (kXAll % kWaves ? 1024 : 0), kSlot = (kRows + (RAW ? 0 : 16 * MT)) * 32;
    static constexpr int kFixed = kScales + 2 * kSlot;
    static_assert(kFixed * per_cu(MT) <= 160 * 1024 && kLoads < 16, "");
};
// RAW: bytes of `rows` quantised rows of `chunks` chunks in LDS, codes and scales.
__host__ __device__ constexpr int resident_bytes(int format, int rows, int chunks) {
    return rows * chunks * ((format == NQX_FP4 ? 128 : 256) + 8);
}

template <typename T, int FORMAT, int MT, bool RAW>
__global__ __launch_bounds__(2 * weight_rows(MT)) void mx_stream_kernel(const void* __restrict__ x, int64_t x_stride, const uint8_t* __restrict__ xs,
                                                             const uint8_t* __restrict__ w, const uint8_t* __restrict__ ws,
                                                             const typename T::elem* __restrict__ bias, typename T::elem* __restrict__ y,
                                                             float* __restrict__ sums, int rows, int N, int blocks, int words, int tiles,
                                                             int splits) {
    using G = Stream<FORMAT, MT, RAW>;
    constexpr bool kFour = FORMAT == NQX_FP4;
    constexpr int kRows = G::kRows, kWaves = G::kWaves, kThreads = G::kThreads, kBufs = G::kBufs;
    extern __shared__ __attribute__((aligned(16))) unsigned char s_mem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lo = lane & 15, hi = lane >> 4;
    const int split = blockIdx.x / tiles, n0 = (blockIdx.x - split * tiles) * kRows;
    const int n_rows = N - n0 < kRows ? N - n0 : kRows;
    const uint32_t w_pitch = (uint32_t)blocks * 16, x_pitch = (uint32_t)blocks * (kFour ? 16 : 32);
    // Chunks: the blocks that do not fill one come first (pieces that do not exist are asked for past the buffer's end, which
    // leaves zeros), then the whole ones.  Scales come for a group of chunks at a time, 32 bytes of a row: for the chunk that is
    // not whole, then for four whole ones each.  A split has whole groups.
    const int part = blocks & 7, whole = blocks >> 3, first = part ? 1 : 0, all_groups = first + ((whole + 3) >> 2);
    const int g0 = (int)((int64_t)all_groups * split / splits), g1 = (int)((int64_t)all_groups * (split + 1) / splits);
    const auto chunk_of = [&](int g) { return g < first ? 0 : min(first + 4 * (g - first), first + whole); };
    const int c0 = chunk_of(g0), c1 = chunk_of(g1);

    const uint8_t *wb = w + (int64_t)n0 * w_pitch, *wsb = ws + (int64_t)n0 * blocks, *xb = static_cast<const uint8_t*>(x);
    const auto buffer = [](const uint8_t* p, uint32_t bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, bytes, 0x00020000);
    };
    const auto bring = [&](__amdgpu_buffer_rsrc_t r, uint32_t v, int to, int from) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(s_mem + to), 16, v,
                                                 __builtin_amdgcn_readfirstlane(from), 0, 0);
    };
    // A load-to-LDS writes 1 KiB in the order of the lanes: eight rows of 128 bytes.  A row's 16-byte pieces are stored at position
    // piece ^ (row / 2 % 8), which spreads the 16 rows of a fragment read over all banks; the swizzle is in the source addresses.
    // Rows past an operand's end are past its buffer's: zeros.
    constexpr uint32_t kNowhere = 0x7FFFFFF0u;       // past the end of every buffer
    const auto swizzle = [](int row, int piece) { return (piece ^ (row >> 1)) & 7; };
    const auto load = [&](int c) {                   // chunk c, or nothing past the last
        const bool there = c < c1, partial = c < first;
        const int at = (c % kBufs) * G::kBuf, f = partial ? whole : c - first;
#pragma unroll
        for (int q = 0; q < G::kWLoads; ++q) {
            const int i = wave + kWaves * q, r = 8 * i + (lane >> 3), piece = swizzle(r, lane & 7);
            bring(buffer(wb, there ? n_rows * w_pitch : 0), partial && piece >= part ? kNowhere : r * w_pitch + piece * 16, at + i * 1024, f * 128);
        }
#pragma unroll
        for (int q = 0; q < G::kXLoads; ++q) {
            const int i = wave + kWaves * q, h = i / (2 * MT), r = 8 * (i % (2 * MT)) + (lane >> 3), piece = swizzle(r, lane & 7);
            const bool mine = i < G::kXAll, none = partial && (kFour ? piece >= part : 8 * h + piece >= 2 * part);
            bring(buffer(xb, there && mine ? rows * x_pitch : 0), none ? kNowhere : r * x_pitch + piece * 16,
                  mine ? at + G::kW + i * 1024 : G::kNone, f * 128 * G::kHalves + h * 128);
        }
    };
    const auto start_of = [&](int g) {               // where the 32 bytes begin: 32 of the row are left at most
        const int at = g < first ? 8 * whole : 32 * (g - first), last = (g < first ? blocks : 8 * whole) - 32;
        return at < last ? at : last < 0 ? 0 : last;
    };
    constexpr int kScaleRows = G::kSlot / 32;
    u32x4 sv[2] = {};
    // Rows of whole words come by load-to-LDS, 32 rows at a time; others, and short ones, through registers, a row a thread.
    const auto ask_scales = [&](int g) {
        if (g >= g1) return;
        const int at = start_of(g), slot = G::kScales + (g & 1) * G::kSlot;
        if (words) {
            for (int i = wave; i < kRows / 32; i += kWaves)
                bring(buffer(wsb, n_rows * blocks), (32 * i + (lane >> 1)) * blocks + (lane & 1) * 16, slot + i * 1024, at);
            if constexpr (!RAW) {
                // 16 rows of x are half a request's: the other lanes' are past the end, and past the slot's rows
                for (int i = wave; i < (16 * MT + 31) / 32; i += kWaves) {
                    const int r = 32 * i + (lane >> 1);
                    if (16 * MT % 32 == 0 || r < 16 * MT)
                        bring(buffer(xs, rows * blocks), r * blocks + (lane & 1) * 16, slot + kRows * 32 + i * 1024, at);
                }
            }
        } else if ((int)threadIdx.x < kScaleRows) {
            const int r = threadIdx.x;
            const uint8_t* from = r < kRows ? wsb + (int64_t)(r < n_rows ? r : n_rows - 1) * blocks
                                            : xs + (int64_t)(r - kRows < rows ? r - kRows : rows - 1) * blocks;
            if (blocks >= 32) {
                __builtin_memcpy(sv, from + at, 32);
            } else {
                uint32_t v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    v[i] = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (4 * i + e < blocks) v[i] |= (uint32_t)from[4 * i + e] << (8 * e);
                }
                sv[0] = u32x4{v[0], v[1], v[2], v[3]}, sv[1] = u32x4{v[4], v[5], v[6], v[7]};
            }
        }
    };
    const auto put_scales = [&](int g) {
        if (words || g >= g1 || (int)threadIdx.x >= kScaleRows) return;
        u32x4* s = reinterpret_cast<u32x4*>(s_mem + G::kScales + (g & 1) * G::kSlot) + 2 * threadIdx.x;
        s[0] = sv[0], s[1] = sv[1];
    };

    f32x4 acc[2][MT];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    ask_scales(g0);
    load(c0);
    if (kBufs == 3) load(c0 + 1);
    const int chunks = c1 - c0, r_bytes = chunks * (kFour ? 128 : 256);      // RAW: of a row's codes in LDS; the scales behind all of them
    unsigned char* s_x = s_mem + G::kFixed;
    unsigned char* s_xs = s_x + rows * r_bytes;
    if constexpr (RAW) {
        // rows x the run of k: a lane eight values, four lanes a block; what is not there becomes zeros
        using E = typename T::elem;
        const int per_row = chunks * 32;
        for (int i = threadIdx.x; i < rows * per_row; i += kThreads) {
            const int r = i / per_row, e = i - r * per_row, c = c0 + (e >> 5);
            const int in_chunk = (e & 31) * 8, at = 256 * (c < first ? whole : c - first) + in_chunk;
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (at < blocks * 32) load8<T>(static_cast<const E*>(x) + r * x_stride + at, v);
            const uint32_t byte = scale_byte<FORMAT>(max_of_block(magnitude_bits(v)));
            const u32x2 code = encode8<FORMAT>(v, byte);
            const int b = in_chunk >> 5, within = in_chunk & 31;               // block of the chunk
            if constexpr (kFour) {
                *reinterpret_cast<uint32_t*>(s_x + r * r_bytes + (c - c0) * 128 + swizzle(r, b) * 16 + within / 2) = code.x;
            } else {
                const int h = b >> 2, piece = (b & 3) * 2 + (within >> 4);
                *reinterpret_cast<u32x2*>(s_x + r * r_bytes + (c - c0) * 256 + h * 128 + swizzle(r, piece) * 16 + (within & 15)) = code;
            }
            if ((e & 3) == 0) s_xs[r * chunks * 8 + (c - c0) * 8 + b] = (unsigned char)byte;
        }
    }
    put_scales(g0);

    const int w_row = wave * 32 + lo, x_own = lo < rows ? lo : rows - 1;
#pragma unroll 1
    for (int c = c0; c < c1; ++c) {
        // chunk c has landed, of three buffers c + 1 may be on its way; nobody needs the buffer of c - 1 any more
        __builtin_amdgcn_s_waitcnt(0x0070 | (kBufs == 3 ? G::kLoads : 0));      // vmcnt(n), lgkmcnt(0)
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        const int g = c < first ? 0 : first + ((c - first) >> 2);
        const bool begins = c == chunk_of(g);
        if (begins) ask_scales(g + 1);
        load(c + kBufs - 1);
        const int at = (c % kBufs) * G::kBuf;
        // where the chunk's scales are in the group's bytes; of the chunk that is not whole a block that is none has zeros for codes
        // and the scale of the last block, which is no NaN unless the row's sum is
        const int s = G::kScales + (g & 1) * G::kSlot + 8 * (c < first ? whole : c - first) - start_of(g), last = c < first ? part - 1 : 7;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int b = 4 * h + hi < last ? 4 * h + hi : last;
            u32x4 a[2];
            uint32_t as[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = w_row + 16 * i;
                a[i] = *reinterpret_cast<const u32x4*>(s_mem + at + r * 128 + swizzle(r, 4 * h + hi) * 16);
                as[i] = s_mem[s + r * 32 + b];
            }
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                u32x4 x0, x1;
                uint32_t bs;
                if constexpr (RAW) {
                    const unsigned char* p = s_x + x_own * r_bytes + (c - c0) * (kFour ? 128 : 256);
                    if constexpr (kFour) {
                        x0 = x1 = *reinterpret_cast<const u32x4*>(p + swizzle(x_own, 4 * h + hi) * 16);
                    } else {
                        x0 = *reinterpret_cast<const u32x4*>(p + h * 128 + swizzle(x_own, hi) * 16);
                        x1 = *reinterpret_cast<const u32x4*>(p + h * 128 + swizzle(x_own, 4 + hi) * 16);
                    }
                    bs = s_xs[x_own * chunks * 8 + (c - c0) * 8 + 4 * h + hi];
                } else {
                    const int r = 16 * j + lo;
                    const unsigned char* p = s_mem + at + G::kW + r * 128;
                    if constexpr (kFour) {
                        x0 = x1 = *reinterpret_cast<const u32x4*>(p + swizzle(r, 4 * h + hi) * 16);
                    } else {
                        x0 = *reinterpret_cast<const u32x4*>(p + h * G::kXHalf + swizzle(r, hi) * 16);
                        x1 = *reinterpret_cast<const u32x4*>(p + h * G::kXHalf + swizzle(r, 4 + hi) * 16);
                    }
                    bs = s_mem[s + (kRows + r) * 32 + b];
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) acc[i][j] = mfma<FORMAT>(a[i], x0, x1, acc[i][j], as[i], bs);
            }
        }
        if (begins) put_scales(g + 1);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);              // vmcnt(0): no request is on its way to LDS that is another workgroup's by then
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int m = 16 * j + lo, n = n0 + wave * 32 + 16 * i + 4 * hi;
            if (m >= rows || n >= N) continue;
            if (splits > 1) *reinterpret_cast<f32x4*>(sums + ((int64_t)split * rows + m) * ((int64_t)tiles * kRows) + n) = acc[i][j];
            else store_sums<T>(acc[i][j], y, bias, m, n, N);
        }
}

// y = the splits' sums, added in order, + bias.
template <typename T>
__global__ __launch_bounds__(256) void mx_add_splits_kernel(const float* __restrict__ sums, const typename T::elem* __restrict__ bias,
                                                            typename T::elem* __restrict__ y, int rows, int N, int pitch, int splits) {
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, n = at % pitch, m = at / pitch;
    if (m >= rows || n >= N) return;
    f32x4 v = *reinterpret_cast<const f32x4*>(sums + at);
    for (int s = 1; s < splits; ++s) v += *reinterpret_cast<const f32x4*>(sums + (int64_t)s * rows * pitch + at);
    store_sums<T>(v, y, bias, m, n, N);
}

template <typename T, int FORMAT, int MT, bool RAW>
hipError_t launch(const Product& p, hipStream_t stream) {
    using G = Stream<FORMAT, MT, RAW>;
    using E = typename T::elem;
    const int blocks = (int)(p.k / kBlock), tiles = (int)cdiv(p.n, G::kRows), splits = stream_splits(p.rows, p.n, p.k, p.format);
    const int chunks = (blocks & 7 ? 1 : 0) + (blocks >> 3);
    const int lds = G::kFixed + (RAW ? resident_bytes(FORMAT, (int)p.rows, stream_chunks(chunks, blocks, splits)) : 0);
    if (lds > 64 * 1024)
        if (const hipError_t e = allow_lds<&mx_stream_kernel<T, FORMAT, MT, RAW>>(160 * 1024); e != hipSuccess) return e;
    const int words = blocks % 4 == 0 && blocks >= 32 && ((reinterpret_cast<uintptr_t>(p.ws) | reinterpret_cast<uintptr_t>(p.xs)) & 3) == 0;
    const E *bias = static_cast<const E*>(p.bias);
    E* y = static_cast<E*>(p.y);
    const hipError_t e = start(&mx_stream_kernel<T, FORMAT, MT, RAW>, dim3(tiles * splits), G::kThreads, lds, stream, RAW ? p.raw : p.x,
                               p.raw_stride, p.xs, p.w, p.ws, bias, y, p.sums, (int)p.rows, (int)p.n, blocks, words, tiles, splits);
    if (e != hipSuccess || splits == 1) return e;
    const int pitch = tiles * G::kRows;
    return start(&mx_add_splits_kernel<T>, dim3((unsigned)cdiv(p.rows * pitch, 1024)), 256, 0, stream, p.sums, bias, y, (int)p.rows, (int)p.n,
                 pitch, splits);
}

}  // namespace

int stream_product(const Product& p, hipStream_t stream) {
    hipError_t e = hipSuccess;
    by_type(p.dtype, p.format, [&](auto t, auto f) {
        using T = decltype(t);
        constexpr int F = decltype(f)::value;
        if (p.raw) e = launch<T, F, 1, true>(p, stream);
        else if (sixteens(p.rows) == 1) e = launch<T, F, 1, false>(p, stream);
        else if (sixteens(p.rows) == 2) e = launch<T, F, 2, false>(p, stream);
        else if (sixteens(p.rows) == 4) e = launch<T, F, 4, false>(p, stream);
        else e = launch<T, F, 8, false>(p, stream);
    });
    return hip_status("mx_stream_kernel", e);
}

// As many splits as fill the chip with workgroups that are resident at once, of a group of chunks each at least.
int stream_splits(int64_t rows, int64_t n, int64_t k, int) {
    const int mt = sixteens(rows);
    const int64_t tiles = cdiv(n, weight_rows(mt)), blocks = k / kBlock, groups = (blocks & 7 ? 1 : 0) + ((blocks >> 3) + 3) / 4;
    int64_t s = 256 * per_cu(mt) / tiles;
    if (s > groups) s = groups;
    if (s > 16) s = 16;
    return s < 1 ? 1 : (int)s;
}
// The most chunks that one of `splits` runs has.
int stream_chunks(int chunks, int blocks, int splits) {
    const int first = blocks & 7 ? 1 : 0, whole = chunks - first, groups = first + (whole + 3) / 4;
    const int most = 4 * (int)cdiv(groups, splits);
    return most < chunks ? most : chunks;
}
size_t stream_sums_bytes(int64_t rows, int64_t n, int64_t k, int format) {
    const int64_t s = stream_splits(rows, n, k, format);
    const int64_t tile = weight_rows(sixteens(rows));
    return s > 1 ? (size_t)(s * rows * cdiv(n, tile) * tile * 4) : 0;
}
int stream_raw_bytes(int64_t rows, int64_t n, int64_t k, int format) {
    const int blocks = (int)(k / kBlock), chunks = (blocks & 7 ? 1 : 0) + (blocks >> 3);
    return resident_bytes(format, (int)rows, stream_chunks(chunks, blocks, stream_splits(rows, n, k, format)));
}

}  // namespace nqx
