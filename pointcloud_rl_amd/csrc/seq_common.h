// Shared by the sequence operators (ssm_*.hip, short_conv.hip, dropout.hip): element types, guarded vector loads, the gates' arithmetic.
#pragma once
#include "common.h"
#include <type_traits>
#include <utility>

namespace pcrl {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

template <int... I, class F>
__device__ __forceinline__ void static_for_impl(std::integer_sequence<int, I...>, F&& f) { (f(std::integral_constant<int, I>{}), ...); }
// f(integral_constant<0>) ... f(integral_constant<N - 1>): for builtins whose operands must be compile-time constants.
template <int N, class F>
__device__ __forceinline__ void static_for(F&& f) { static_for_impl(std::make_integer_sequence<int, N>{}, f); }

// V consecutive elements as they stand in memory, so that a load can stay in flight until its first use.
template <typename T, int V>
struct RawVec { T v[V]; };
template <typename T, int V>
__device__ __forceinline__ RawVec<T, V> raw_zero() {
    RawVec<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = (T)0.0f;
    return r;
}
// n: how many of the V elements exist (<= 0: none, nothing is read).  vec: the address is aligned to the whole vector and n is 0 or V.
template <typename T, int V>
__device__ __forceinline__ RawVec<T, V> raw_load(const T* p, int n, bool vec) {
    typedef T vt __attribute__((ext_vector_type(V)));
    RawVec<T, V> r = raw_zero<T, V>();
    if (n > 0) {
        if (vec) {
            const vt x = *(const vt*)p;
#pragma unroll
            for (int i = 0; i < V; ++i) r.v[i] = x[i];
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) if (i < n) r.v[i] = p[i];
        }
    }
    return r;
}
// One rounding to the element type (round to nearest even): the only rounding between the 32-bit sums and memory.
template <typename T, int V>
__device__ __forceinline__ void raw_store(T* p, const float (&x)[V], int n, bool vec) {
    typedef T vt __attribute__((ext_vector_type(V)));
    if (n <= 0) return;
    if (vec) {
        vt y;
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = (T)x[i];
        *(vt*)p = y;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) if (i < n) p[i] = (T)x[i];
    }
}

__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
// 1 / (1 + exp(-x)): 0 and 1 at the ends, NaN stays NaN.
__device__ __forceinline__ float sigmoidf_(float x) { return __builtin_amdgcn_rcpf(1.0f + fast_exp(-x)); }
// log(1 + exp(x)) and its derivative.  log1p(e) for e in [0, 1] is log(w) + (e - (w - 1)) / w with w = 1 + e rounded: the second term puts the
// rounding of 1 + e back, so the result keeps full relative precision where softplus is small.
__device__ __forceinline__ float softplus_(float x, float& slope) {
    const float e = fast_exp(-__builtin_fabsf(x)), w = 1.0f + e, r = __builtin_amdgcn_rcpf(w);
    slope = x >= 0.0f ? r : e * r;
    return __builtin_fmaxf(x, 0.0f) + __builtin_fmaf(e - (w - 1.0f), r, __builtin_amdgcn_logf(w) * kLn2);
}

// V adjacent elements at a base that is the same for the whole wave + a 32-bit element offset per lane (one address register per lane instead of
// two, no 64-bit sums), or, VEC false, each at an offset of its own.  The caller clamps the offsets to what exists.
template <typename T, int V, bool VEC>
__device__ __forceinline__ RawVec<T, V> lane_load(const T* base, unsigned row, const unsigned (&at)[V]) {
    RawVec<T, V> r;
    if constexpr (VEC && V > 1) {
        typedef T vt __attribute__((ext_vector_type(V)));
        const vt x = *(const vt*)((const char*)base + (row + at[0]) * (unsigned)sizeof(T));
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = x[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = *(const T*)((const char*)base + (row + at[i]) * (unsigned)sizeof(T));
    }
    return r;
}
// n: how many of the V elements exist; VEC: all or none.
template <typename T, int V, bool VEC>
__device__ __forceinline__ void lane_store(T* base, unsigned off, const float (&x)[V], int n) {
    if constexpr (VEC && V > 1) {
        typedef T vt __attribute__((ext_vector_type(V)));
        vt y;
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = (T)x[i];
        if (n > 0) *(vt*)((char*)base + off * (unsigned)sizeof(T)) = y;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) if (i < n) *(T*)((char*)base + (off + i) * (unsigned)sizeof(T)) = (T)x[i];
    }
}

// Lane I of each row of 16 lanes, in every lane of that row (a DPP operand of the instruction that uses it).
template <int I>
__device__ __forceinline__ float row_bcast(float v) {
    return u2f((unsigned)__builtin_amdgcn_update_dpp(0, (int)f2u(v), 0x150 + I, 0xF, 0xF, true));
}

// acc[j] += (lane I of the row of c[j]) * x, and the sum over j of (lane I of the row of c[j]) * x[j].  The compiler folds a row broadcast into a
// multiply but not into a multiply-add.  s_nop 1: the two wait states between a vector instruction that may have written c and the DPP read of
// it, whatever stands in front.
#define PCRL_FMAC_ROW(ACC, C, X, I) "v_fmac_f32_dpp %" #ACC ", %" #C ", %" #X " row_newbcast:%" #I " row_mask:0xf bank_mask:0xf\n\t"
template <int I, int RN>
__device__ __forceinline__ void fma_row_bcast(float (&acc)[RN], const float (&c)[RN], float x) {
    if constexpr (RN == 4)
        asm("s_nop 1\n\t" PCRL_FMAC_ROW(0, 4, 8, 9) PCRL_FMAC_ROW(1, 5, 8, 9) PCRL_FMAC_ROW(2, 6, 8, 9) PCRL_FMAC_ROW(3, 7, 8, 9)
            : "+v"(acc[0]), "+v"(acc[1]), "+v"(acc[2]), "+v"(acc[3]) : "v"(c[0]), "v"(c[1]), "v"(c[2]), "v"(c[3]), "v"(x), "n"(I));
    else if constexpr (RN == 2)
        asm("s_nop 1\n\t" PCRL_FMAC_ROW(0, 2, 4, 5) PCRL_FMAC_ROW(1, 3, 4, 5) : "+v"(acc[0]), "+v"(acc[1]) : "v"(c[0]), "v"(c[1]), "v"(x), "n"(I));
    else
        asm("s_nop 1\n\t" PCRL_FMAC_ROW(0, 1, 2, 3) : "+v"(acc[0]) : "v"(c[0]), "v"(x), "n"(I));
}
template <int I, int RN>
__device__ __forceinline__ float dot_row_bcast(const float (&c)[RN], const float (&x)[RN]) {
    float acc = x[0] * row_bcast<I>(c[0]);
    if constexpr (RN == 4)
        asm("s_nop 1\n\t" PCRL_FMAC_ROW(0, 1, 4, 7) PCRL_FMAC_ROW(0, 2, 5, 7) PCRL_FMAC_ROW(0, 3, 6, 7)
            : "+v"(acc) : "v"(c[1]), "v"(c[2]), "v"(c[3]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "n"(I));
    else if constexpr (RN == 2)
        asm("s_nop 1\n\t" PCRL_FMAC_ROW(0, 1, 2, 3) : "+v"(acc) : "v"(c[1]), "v"(x[1]), "n"(I));
    return acc;
}
#undef PCRL_FMAC_ROW

constexpr long long kMaxGroups = (1LL << 24) - 1;      // workgroups of 256: a grid holds fewer than 2^32 threads
__host__ inline int elem_bytes(int dtype) { return dtype == PCRL_DT_F32 ? 4 : 2; }
// Two ranges of memory touch each other without being the same one (same: also when they are).
__host__ inline bool overlap(const void* a, const void* b, size_t bytes, bool same) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && (x != y ? (x < y ? y - x : x - y) < bytes : same);
}
__host__ inline bool seq_dtype(int dtype) { return dtype == PCRL_DT_F32 || dtype == PCRL_DT_BF16 || dtype == PCRL_DT_F16; }

}  // namespace pcrl
