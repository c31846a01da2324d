// Dropout from a counter-based generator (include/pcrl.h: which word decides which element).  The mask is a function of (seed, offset, element
// index), so nothing is stored for the backward: it is the same launch on the gradient.
// One Philox call decides eight elements (16 bits each: probabilities in steps of 2^-16), which is one 16-byte access of a 16-bit type.
// All of it is 173 instructions for eight elements (11 us of every SIMD at 8192 x 2048), so memory bounds it: bf16, 13.4 us without a residual
// (67 MB, 5.0 TB/s) and 17.7 us with one (101 MB, 5.7 TB/s, part of it from the last-level cache).
#include "seq_common.h"

namespace pcrl {

struct DropoutParams {
    const void *x, *residual;
    void* out;
    long long x_ld, residual_ld, rows, cols, n;
    unsigned threshold, seed_lo, seed_hi;
    unsigned long long offset;
    const unsigned long long* offset_ptr;
    float scale;
    int flat;                                          // x, residual and out are dense and aligned: eight elements are one vector
};

template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(const DropoutParams p) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, e0 = i * 8;
    if (e0 >= p.n) return;
    const unsigned long long off = p.offset_ptr ? p.offset_ptr[0] : p.offset;
    const int left = p.n - e0 < 8 ? (int)(p.n - e0) : 8;
    const T *px = (const T*)p.x, *pr = (const T*)p.residual;
    RawVec<T, 8> x, res;
    if (p.flat) {
        x = raw_load<T, 8>(px + e0, left, left == 8);
        res = raw_load<T, 8>(pr ? pr + e0 : px, pr ? left : 0, left == 8);
    } else {
        x = raw_zero<T, 8>(), res = raw_zero<T, 8>();
        long long row = e0 / p.cols, col = e0 - row * p.cols;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (k < left) {
                x.v[k] = px[row * p.x_ld + col];
                if (pr) res.v[k] = pr[row * p.residual_ld + col];
            }
            if (++col == p.cols) { col = 0; ++row; }
        }
    }
    uint32_t w[4];
    philox4x32_10((uint32_t)i, (uint32_t)((unsigned long long)i >> 32), (uint32_t)off, (uint32_t)(off >> 32), p.seed_lo, p.seed_hi, w);
    float y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const unsigned half = (k & 1) ? w[k >> 1] >> 16 : w[k >> 1] & 0xFFFFu;
        const float v = half >= p.threshold ? (float)x.v[k] * p.scale : 0.0f;
        y[k] = pr ? v + (float)res.v[k] : v;
    }
    raw_store<T, 8>((T*)p.out + e0, y, left, p.flat && left == 8);
}

}  // namespace pcrl

using namespace pcrl;

extern "C" int pcrl_dropout(const void* x, int64_t x_ld, const void* residual, int64_t residual_ld, void* out, int64_t rows, int64_t cols, int32_t dtype,
                            int32_t threshold, uint64_t seed, uint64_t offset, const uint64_t* offset_ptr, void* stream) {
    if (!x || !out) return fail(PCRL_E_ARG, "pcrl_dropout: null tensor");
    if (rows < 1 || cols < 1) return fail(PCRL_E_ARG, "pcrl_dropout: %lld x %lld elements", (long long)rows, (long long)cols);
    if (!seq_dtype(dtype)) return fail(PCRL_E_ARG, "pcrl_dropout: dtype %d", dtype);
    if (threshold < 0 || threshold > 65536) return fail(PCRL_E_ARG, "pcrl_dropout: threshold %d", threshold);
    if (rows > (1LL << 40) / cols) return fail(PCRL_E_ARG, "pcrl_dropout: too many elements");
    DropoutParams p{};
    p.x = x, p.residual = residual, p.out = out;
    p.x_ld = x_ld, p.residual_ld = residual_ld, p.rows = rows, p.cols = cols, p.n = rows * cols;
    p.threshold = (unsigned)threshold, p.seed_lo = (unsigned)seed, p.seed_hi = (unsigned)(seed >> 32);
    p.offset = offset, p.offset_ptr = (const unsigned long long*)offset_ptr;
    p.scale = threshold == 65536 ? 0.0f : 65536.0f / (float)(65536 - threshold);
    const size_t bytes = 8 * (size_t)elem_bytes(dtype);
    const size_t align = bytes > 16 ? 16 : bytes;
    p.flat = (x_ld == cols || rows == 1) && (!residual || residual_ld == cols || rows == 1) &&
             ((uintptr_t)x | (uintptr_t)out | (uintptr_t)residual) % align == 0;
    const long long groups = (p.n + 7) / 8, blocks = (groups + 255) / 256;
    if (blocks > kMaxGroups) return fail(PCRL_E_ARG, "pcrl_dropout: too many workgroups");
    const dim3 grid((unsigned)blocks);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == PCRL_DT_F32) dropout_kernel<float><<<grid, 256, 0, s>>>(p);
    else if (dtype == PCRL_DT_BF16) dropout_kernel<__bf16><<<grid, 256, 0, s>>>(p);
    else dropout_kernel<_Float16><<<grid, 256, 0, s>>>(p);
    PCRL_CHECK_LAUNCH("dropout_kernel");
    return PCRL_OK;
}
