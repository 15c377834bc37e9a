// Error plumbing and argument checks of libnq_mx.so.
#include <cstdarg>
#include <cstdio>

#include "mx_common.hpp"

namespace nqx {
namespace {
thread_local char g_error[512] = "";
}

int refuse(int status, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof g_error, fmt, ap);
    va_end(ap);
    return status;
}

int hip_status(const char* fn, hipError_t e) {
    return e == hipSuccess ? NQX_OK : refuse(NQX_ERR_HIP, "%s: HIP error %d (%s)", fn, (int)e, hipGetErrorString(e));
}

int check_types(const char* fn, int64_t rows, int64_t k, int dtype, int format) {
    if (dtype != NQX_F16 && dtype != NQX_BF16 && dtype != NQX_F32)
        return refuse(NQX_ERR_ARG, "%s: dtype must be NQX_F16 (0), NQX_BF16 (1) or NQX_F32 (2), got %d", fn, dtype);
    if (format != NQX_FP4 && format != NQX_FP8)
        return refuse(NQX_ERR_ARG, "%s: format must be NQX_FP4 (0) or NQX_FP8 (1), got %d", fn, format);
    if (rows < 0 || k <= 0 || k % kBlock != 0)
        return refuse(NQX_ERR_ARG, "%s: rows must not be negative and k a positive multiple of %d (rows=%lld k=%lld)", fn, kBlock,
                      (long long)rows, (long long)k);
    // 2^36 values less one workgroup's: a launch has fewer than 2^32 threads along x in whole workgroups of 256, and a thread has 16
    // values at least, half a block
    if (k > ((int64_t)1 << 30) || rows > ((int64_t)1 << 31) || rows * (k / kBlock) > ((int64_t)1 << 31) - 128)
        return refuse(NQX_ERR_UNSUPPORTED, "%s: problem too large (rows=%lld k=%lld)", fn, (long long)rows, (long long)k);
    return NQX_OK;
}

int check_rows(const char* fn, const char* what, const void* p, int64_t stride, int64_t k, int dtype) {
    if (!p || !aligned16(p)) return refuse(NQX_ERR_ARG, "%s: %s must be a 16-byte aligned device pointer", fn, what);
    if (stride < 0 || stride > ((int64_t)1 << 40) || stride * elem_bytes(dtype) % 16 != 0)
        return refuse(NQX_ERR_ARG, "%s: rows of %s must start on 16-byte boundaries (stride %lld)", fn, what, (long long)stride);
    return NQX_OK;
}

}  // namespace nqx

extern "C" const char* nqx_last_error(void) { return nqx::g_error; }
