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
// log(1 + exp(x)) and its derivative.  log1p(e) for e in (0, 1] is log(1 + e) * e / ((1 + e) - 1): the rounding of 1 + e cancels, so the
// result keeps full relative precision where softplus is small.
__device__ __forceinline__ float softplus_(float x, float& slope) {
    const float e = fast_exp(-__builtin_fabsf(x)), w = 1.0f + e, d = w - 1.0f, r = __builtin_amdgcn_rcpf(w);
    const float l = d == 0.0f ? e : __builtin_amdgcn_logf(w) * kLn2 * (e * __builtin_amdgcn_rcpf(d));
    slope = x >= 0.0f ? r : e * r;
    slope = x != x ? x : slope;
    return __builtin_fmaxf(x, 0.0f) + (x != x ? x : l);
}

// Lane I of each row of 16 lanes, in every lane of that row (a DPP operand of the instruction that uses it).
template <int I>
__device__ __forceinline__ float row_bcast(float v) {
    return u2f((unsigned)__builtin_amdgcn_update_dpp(0, (int)f2u(v), 0x150 + I, 0xF, 0xF, true));
}

__host__ inline int elem_bytes(int dtype) { return dtype == PCRL_DT_F32 ? 4 : 2; }
__host__ inline bool seq_dtype(int dtype) { return dtype == PCRL_DT_F32 || dtype == PCRL_DT_BF16 || dtype == PCRL_DT_F16; }

}  // namespace pcrl
