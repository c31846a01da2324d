// Short causal convolution over time, one filter of W taps per channel, optional SiLU (include/pcrl.h: the formulas).
// Bound by memory: a thread owns V adjacent channels (16 bytes) and a run of steps, keeps the last W - 1 inputs in registers and so reads every
// input once (plus W - 1 rows of halo per run).  4 x 2048 x 2048, W = 4, bf16: forward 16.5 us (67 MB, 4.1 TB/s; 11 us of every SIMD are vector
// instructions), backward 27.3 us (101 MB, 3.7 TB/s; 15 us of them, at three waves per SIMD) and 4 us of sums.
#include "seq_common.h"

namespace pcrl {

constexpr int kConvV = 4;                              // adjacent channels of a thread
constexpr int kRun = 8;                                // steps a forward thread takes (16: 18.9 us for 17.4, half the waves)

struct ConvParams {
    int B, T, D, silu, vec, vec_w, nrun, run;          // vec, vec_w: whole vectors of the activations, of the weights; runs of `run` steps (backward)
    long long x_sb, x_st, dy_sb, dy_st, starts_sb;
    const void *x, *state, *dy, *dlast;
    const float *weight, *bias;
    const uint8_t* starts;
    const int* lengths;
    void *y, *last, *dx, *dstate;
    float* part;                                       // [parts][W + 1][D]: dweight by tap, then dbias
    int parts;
};

__device__ __forceinline__ int conv_length(const ConvParams& p, int b) {
    if (!p.lengths) return p.T;
    const int n = p.lengths[b];
    return n < 0 ? 0 : n > p.T ? p.T : n;
}

// Inputs of the W - 1 steps in front of step t (what of them belongs to t's sequence, state rows where t is near the front), oldest first.
template <typename T, int V, int W>
__device__ __forceinline__ void conv_window(const ConvParams& p, int b, int d0, int nv, int t, float (&win)[W][V]) {
    const T* px = (const T*)p.x + b * p.x_sb + d0;
    const T* ps = p.state ? (const T*)p.state + (long long)b * (W - 1) * p.D + d0 : nullptr;
    RawVec<T, V> raw[W];
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
        const int s = t - (W - 1) + k;
        raw[k] = s >= 0 ? raw_load<T, V>(px + s * p.x_st, nv, p.vec) : raw_load<T, V>(ps ? ps + (s + W - 1) * (long long)p.D : px, ps ? nv : 0, p.vec);
    }
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) win[k][i] = (float)raw[k].v[i];
    if (p.starts) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {              // a start at step s cuts off everything older
            const int s = t - (W - 1) + k;
            if (s >= 0 && p.starts[b * p.starts_sb + s])
#pragma unroll
                for (int j = 0; j < k; ++j)
#pragma unroll
                    for (int i = 0; i < V; ++i) win[j][i] = 0.0f;
        }
    }
}

// The W taps of the thread's channels: V W adjacent floats.
template <int V, int W>
__device__ __forceinline__ void conv_weights(const ConvParams& p, int d0, int nv, float (&w)[W][V], float (&bias)[V]) {
    if (p.vec_w && nv == V) {
        const f32x4* src = (const f32x4*)(p.weight + (long long)d0 * W);
        float flat[V * W];
#pragma unroll
        for (int e = 0; e < V * W / 4; ++e) {
            const f32x4 x = src[e];
#pragma unroll
            for (int i = 0; i < 4; ++i) flat[4 * e + i] = x[i];
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int k = 0; k < W; ++k) w[k][i] = flat[i * W + k];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int k = 0; k < W; ++k) w[k][i] = i < nv ? p.weight[(long long)(d0 + i) * W + k] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = i < nv && p.bias ? p.bias[d0 + i] : 0.0f;
}

template <typename T, int V, int W>
__global__ __launch_bounds__(256) void conv_fwd_kernel(const ConvParams p) {
    // Workgroups go to the eight XCDs in turn: dealt out so that each XCD has adjacent runs, whose halo rows are then in its own L2
    // (17.2 -> 16.5 us).
    const unsigned xcd = blockIdx.x & 7u, some = gridDim.x >> 3, more = gridDim.x & 7u;
    const unsigned blk = xcd * some + (xcd < more ? xcd : more) + (blockIdx.x >> 3);
    const unsigned nvec = (unsigned)(p.D + V - 1) / V, runs = (unsigned)p.nrun + 1;      // (a grid holds fewer than 2^32 threads: 32-bit divisions)
    const unsigned idx = blk * 256u + threadIdx.x, line = idx / nvec;
    const int d0 = (int)(idx - line * nvec) * V, nv = p.D - d0 < V ? p.D - d0 : V;
    const int b = (int)(line / runs), q = (int)(line - (unsigned)b * runs);
    if (b >= p.B) return;
    const int len = conv_length(p, b);
    float win[W][V];
    if (q == p.nrun) {                                 // the state after the last step
        if (!p.last || W == 1) return;
        conv_window<T, V, W>(p, b, d0, nv, len, win);
#pragma unroll
        for (int k = 0; k < W - 1; ++k) raw_store<T, V>((T*)p.last + ((long long)b * (W - 1) + k) * p.D + d0, win[k], nv, p.vec);
        return;
    }
    float w[W][V], bias[V];
    conv_weights<V, W>(p, d0, nv, w, bias);
    const int t_first = q * kRun, t_last = t_first + kRun < p.T ? t_first + kRun : p.T;
    const T* px = (const T*)p.x + b * p.x_sb + d0;
    T* py = (T*)p.y + (long long)b * p.T * p.D + d0;
    RawVec<T, V> raw[kRun];                            // the whole run in flight, the window's rows with it
    bool st[kRun];
    // Almost every wave: all rows exist and no start is near (one test for the wave, then nothing but loads).
    const bool easy = p.vec && !p.starts && t_first >= W - 1 && t_first + kRun <= len;
    if (__all(easy)) {
        RawVec<T, V> before[W];
#pragma unroll
        for (int k = 0; k < W - 1; ++k) before[k] = raw_load<T, V>(px + (long long)(t_first - (W - 1) + k) * p.x_st, V, true);
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            raw[k] = raw_load<T, V>(px + (long long)(t_first + k) * p.x_st, V, true);
            st[k] = false;
        }
#pragma unroll
        for (int k = 0; k < W - 1; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) win[k][i] = (float)before[k].v[i];
    } else {
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            const int t = t_first + k;
            const bool on = t < t_last && t < len;
            raw[k] = raw_load<T, V>(px + (long long)t * p.x_st, on ? nv : 0, p.vec);
            st[k] = p.starts && on && p.starts[b * p.starts_sb + t];
        }
        conv_window<T, V, W>(p, b, d0, t_first < len ? nv : 0, t_first, win);
    }
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
        const int t = t_first + k;
        float out[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (st[k])
#pragma unroll
                for (int j = 0; j < W - 1; ++j) win[j][i] = 0.0f;
            win[W - 1][i] = (float)raw[k].v[i];
            float acc = bias[i];
#pragma unroll
            for (int j = 0; j < W; ++j) acc = __builtin_fmaf(w[j][i], win[j][i], acc);
            out[i] = acc;
#pragma unroll
            for (int j = 0; j < W - 1; ++j) win[j][i] = win[j + 1][i];
        }
        if (p.silu) {
#pragma unroll
            for (int i = 0; i < V; ++i) out[i] *= sigmoidf_(out[i]);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = t < len ? out[i] : 0.0f;
        raw_store<T, V>(py + (long long)t * p.D, out, t < t_last ? nv : 0, p.vec);
    }
}

// One step: a thread reads the W - 1 state rows of its channels before it writes them, so the state may be updated in place.  5.0 us at 64 x 512,
// W = 4, float32, of which a launch is 2.7: its weights come as single conditional loads.
template <typename T, int V, int W>
__global__ __launch_bounds__(256) void conv_step_kernel(const ConvParams p) {
    const unsigned nvec = (unsigned)(p.D + V - 1) / V, idx = blockIdx.x * 256u + threadIdx.x, line = idx / nvec;
    if (line >= (unsigned)p.B) return;
    const int b = (int)line, d0 = (int)(idx - line * nvec) * V, nv = p.D - d0 < V ? p.D - d0 : V;
    const bool on = conv_length(p, b) > 0;
    const RawVec<T, V> raw = raw_load<T, V>((const T*)p.x + b * p.x_sb + d0, on ? nv : 0, p.vec);
    float win[W][V];
    conv_window<T, V, W>(p, b, d0, nv, 0, win);
    const bool st = on && p.starts && p.starts[b * p.starts_sb];
    float out[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) win[j][i] = st ? 0.0f : win[j][i];
        win[W - 1][i] = (float)raw.v[i];
        float acc = i < nv && p.bias ? p.bias[d0 + i] : 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) acc = __builtin_fmaf(i < nv ? p.weight[(long long)(d0 + i) * W + j] : 0.0f, win[j][i], acc);
        if (p.silu) acc *= sigmoidf_(acc);
        out[i] = on ? acc : 0.0f;
    }
    raw_store<T, V>((T*)p.y + (long long)b * p.D + d0, out, nv, p.vec);
    if (p.last) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
            if (on) raw_store<T, V>((T*)p.last + ((long long)b * (W - 1) + k) * p.D + d0, win[k + 1], nv, p.vec);
            else raw_store<T, V>((T*)p.last + ((long long)b * (W - 1) + k) * p.D + d0, win[k], nv, p.vec);
        }
    }
}

// Backward.  A thread walks its run (and W - 1 steps behind it, whose outputs its inputs also feed): dpre of step s from the window of inputs,
// then dx of the last W inputs gets its tap's share.  An input is complete when its W-th step has passed or a new sequence has begun.
// Steps without tests (whole vectors, no starts) have a body of their own: 40.8 -> 29.3 us; runs of 32 instead of 16: 27.3 (of 8: 35).  A fourth
// wave per SIMD (128 registers) spills: 38; the next group's loads ahead of this one's arithmetic: 25.9, but 12.2 -> 13.1 at 256 x 16 x 256.
template <typename T, int V, int W>
__global__ __launch_bounds__(256) void conv_bwd_kernel(const ConvParams p) {
    extern __shared__ float s_part[];                  // [4][W + 1][64 V]
    // a workgroup: 64 channel vectors x 4 walkers; walker (blockIdx.y, k) takes every parts-th (b, run)
    const int lane = threadIdx.x & 63, k4 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int d0 = (blockIdx.x * 64 + lane) * V, nv = p.D - d0 < V ? p.D - d0 : V;       // nv <= 0: no channel
    const unsigned lanes[V] = {nv > 0 ? (unsigned)d0 : 0u};             // (whole vectors only: the first element's place)
    float w[W][V], bias[V], dw[W][V], db[V];
    conv_weights<V, W>(p, d0, nv, w, bias);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        db[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) dw[k][i] = 0.0f;
    }
    const long long lines = (long long)p.B * p.nrun;
    for (long long line = (long long)blockIdx.y * 4 + k4; line < lines; line += 4LL * p.parts) {
        const int b = (int)(line / p.nrun), q = (int)(line - (long long)b * p.nrun);
        const int len = conv_length(p, b);
        const int t_first = q * p.run, t_last = t_first + p.run < p.T ? t_first + p.run : p.T;
        const T* px = (const T*)p.x + b * p.x_sb;
        const T* pg = (const T*)p.dy + b * p.dy_sb;
        const uint8_t* ps = p.starts ? p.starts + b * p.starts_sb : nullptr;
        T* dx = (T*)p.dx + (long long)b * p.T * p.D;
        float win[W][V], acc[W][V];                    // inputs s - (W - 1) ... s and their dx so far
        bool alive[W];                                 // ... still in the sequence of step s
#pragma unroll
        for (int j = 0; j < W; ++j) {
            alive[j] = true;
#pragma unroll
            for (int i = 0; i < V; ++i) win[j][i] = acc[j][i] = 0.0f;
        }
        if (W > 1) conv_window<T, V, W>(p, b, d0, nv, t_first, win);
        auto finish = [&](int t, const float (&g)[V]) __attribute__((always_inline)) {              // dx of input t is complete
            if (t >= t_first && t < t_last) {
                if (p.vec) lane_store<T, V, true>(dx + (long long)t * p.D, (unsigned)d0, g, nv);
                else lane_store<T, V, false>(dx + (long long)t * p.D, (unsigned)d0, g, nv);
            }
            else if (t < 0 && q == 0 && p.dstate) raw_store<T, V>((T*)p.dstate + ((long long)b * (W - 1) + t + W - 1) * p.D + d0, g, nv, p.vec);
        };
        // taps that a start before t_first cut off from the state: their rows get no gradient (they stay zero); inside the run `alive` says so
        const int stop = t_last + W - 1 < len ? t_last + W - 1 : len;           // steps walked: [t_first, stop)
        constexpr int U = 4;
        // One group of U steps from s0 on.  EASY: whole vectors and no starts; OWN: steps of this run (the ones behind it give no share of dweight and
        // dbias here); FULL: all U steps are before `to`.  All of it uniform over the wave.
        auto group = [&](auto easy_, auto own_, auto full_, int s0, int to) __attribute__((always_inline)) {
            constexpr bool EASY = decltype(easy_)::value, STARTS = !EASY, OWN = decltype(own_)::value, FULL = decltype(full_)::value;
            RawVec<T, V> rx[U], rg[U];
            bool st[U];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const bool on = FULL || s0 + k < to;
                if constexpr (EASY) {                  // (rows behind the last one of the group read it again)
                    const long long row = on ? s0 + k : to - 1;
                    rx[k] = lane_load<T, V, true>(px + row * p.x_st, 0, lanes);
                    rg[k] = lane_load<T, V, true>(pg + row * p.dy_st, 0, lanes);
                } else {
                    rx[k] = raw_load<T, V>(px + (long long)(s0 + k) * p.x_st + d0, on ? nv : 0, p.vec);
                    rg[k] = raw_load<T, V>(pg + (long long)(s0 + k) * p.dy_st + d0, on ? nv : 0, p.vec);
                }
                st[k] = STARTS && ps && on && ps[s0 + k];
            }
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int s = s0 + k;
                if (!FULL && s >= to) break;
                if (STARTS && st[k]) {
#pragma unroll
                    for (int j = 0; j < W - 1; ++j) alive[j] = false;
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (STARTS && st[k])
#pragma unroll
                        for (int j = 0; j < W - 1; ++j) win[j][i] = 0.0f;
                    win[W - 1][i] = (float)rx[k].v[i];
                    acc[W - 1][i] = 0.0f;
                    float dpre = (float)rg[k].v[i];
                    if (p.silu) {
                        float pre = bias[i];
#pragma unroll
                        for (int j = 0; j < W; ++j) pre = __builtin_fmaf(w[j][i], win[j][i], pre);
                        const float sg = sigmoidf_(pre);
                        dpre *= __builtin_fmaf(pre * sg, 1.0f - sg, sg);
                    }
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        if (!STARTS || j == W - 1 || alive[j]) acc[j][i] = __builtin_fmaf(w[j][i], dpre, acc[j][i]);
                        if (OWN) dw[j][i] = __builtin_fmaf(dpre, win[j][i], dw[j][i]);
                    }
                    if (OWN) db[i] += dpre;
                }
                finish(s - (W - 1), acc[0]);
#pragma unroll
                for (int j = 0; j < W - 1; ++j) {
                    if (STARTS) alive[j] = j + 1 < W - 1 ? alive[j + 1] : true;
#pragma unroll
                    for (int i = 0; i < V; ++i) { win[j][i] = win[j + 1][i]; acc[j][i] = acc[j + 1][i]; }
                }
            }
        };
        auto walk = [&](auto easy) __attribute__((always_inline)) {
            const std::true_type yes;
            const std::false_type no;
            const int mid = t_last < stop ? t_last : stop;
            int s0 = t_first;
            for (; s0 + U <= mid; s0 += U) group(easy, yes, easy, s0, mid);
            if (s0 < mid) group(easy, yes, no, s0, mid);
            if (W > 1 && mid < stop) group(easy, no, no, mid, stop);
        };
        if (p.vec && !ps) walk(std::true_type{});
        else walk(std::false_type{});
        // what is left in the window: inputs at - (W - 1) ... at - 1, where `at` is the step behind the last walked one
        const int at = stop > t_first ? stop : t_first;
        if (at <= len || q == 0) {
#pragma unroll
            for (int j = 0; j < W - 1; ++j) {
                const int t = at - (W - 1) + j;
                float gl[V];
#pragma unroll
                for (int i = 0; i < V; ++i) gl[i] = acc[j][i];
                if (at == len && alive[j] && p.dlast) {               // it stands in the last state: row j
                    const RawVec<T, V> dl = raw_load<T, V>((const T*)p.dlast + ((long long)b * (W - 1) + j) * p.D + d0, nv, p.vec);
#pragma unroll
                    for (int i = 0; i < V; ++i) gl[i] += (float)dl.v[i];
                }
                if (t < len) finish(t, gl);
            }
        }
        float none[V];
#pragma unroll
        for (int i = 0; i < V; ++i) none[i] = 0.0f;
        for (int t = t_first > len ? t_first : len; t < t_last; ++t) raw_store<T, V>(dx + (long long)t * p.D + d0, none, nv, p.vec);
    }
    // the four walkers' sums, in order
#pragma unroll
    for (int j = 0; j < W + 1; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) s_part[(k4 * (W + 1) + j) * (64 * V) + lane * V + i] = j < W ? dw[j < W ? j : 0][i] : db[i];
    __syncthreads();
    for (int e = threadIdx.x; e < (W + 1) * 64 * V; e += 256) {
        const int j = e / (64 * V), c = e - j * (64 * V), d = blockIdx.x * 64 * V + c;
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) t += s_part[(k * (W + 1) + j) * (64 * V) + c];
        if (d < p.D) p.part[((long long)blockIdx.y * (W + 1) + j) * p.D + d] = t;
    }
}

// dweight [D][W] and dbias [D]: the parts, in order; 16 threads a channel.
__global__ __launch_bounds__(1024) void conv_finish_kernel(const float* part, int parts, int W, int D, float* dweight, float* dbias) {
    __shared__ float s_sum[16][64];
    const int j = blockIdx.y, d = blockIdx.x * 64 + (threadIdx.x & 63), k = threadIdx.x >> 6;
    float sum = 0.0f;
    if (d < D) {
#pragma unroll 8
        for (int i = k; i < parts; i += 16) sum += part[((long long)i * (W + 1) + j) * D + d];
    }
    s_sum[k][threadIdx.x & 63] = sum;
    __syncthreads();
    if (threadIdx.x < 64 && d < D) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += s_sum[i][threadIdx.x];
        if (j < W) dweight[(long long)d * W + j] = t;
        else if (dbias) dbias[d] = t;
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------
static int conv_check(const pcrl_conv_desc* d, const char* who) {
    if (!d) return fail(PCRL_E_ARG, "%s: null descriptor", who);
    if (d->B < 1 || d->T < 1 || d->D < 1) return fail(PCRL_E_ARG, "%s: B, T, D must be positive (%d, %d, %d)", who, d->B, d->T, d->D);
    if (d->T > 0x7FFFFFE0 || d->D >= (1 << 26)) return fail(PCRL_E_ARG, "%s: T = %d, D = %d", who, d->T, d->D);        // (32-bit steps and channels)
    if (d->W < 1 || d->W > 4) return fail(PCRL_E_ARG, "%s: W = %d taps (1 to 4)", who, d->W);
    if (!seq_dtype(d->dtype)) return fail(PCRL_E_ARG, "%s: dtype %d", who, d->dtype);
    if (!d->x || !d->weight) return fail(PCRL_E_ARG, "%s: null input", who);
    return PCRL_OK;
}
static void conv_fill(ConvParams& p, const pcrl_conv_desc* d) {
    p = ConvParams{};
    p.B = d->B, p.T = d->T, p.D = d->D, p.silu = d->silu != 0;
    p.x = d->x, p.x_sb = d->x_sb, p.x_st = d->x_st, p.weight = d->weight, p.bias = d->bias, p.state = d->state;
    p.starts = d->starts, p.starts_sb = d->starts_sb, p.lengths = d->lengths;
    p.vec_w = (uintptr_t)d->weight % 16 == 0;
}
static bool conv_vec(const pcrl_conv_desc* d, int V, const void* const* extra, int n) {
    const size_t bytes = (size_t)V * elem_bytes(d->dtype);
    if (d->D % V || d->x_sb % V || d->x_st % V || (uintptr_t)d->x % bytes || (uintptr_t)d->state % bytes) return false;
    for (int i = 0; i < n; ++i) if ((uintptr_t)extra[i] % bytes) return false;
    return true;
}

template <typename T, int V, int W>
static int conv_fwd(ConvParams& p, hipStream_t s) {
    const long long nvec = (p.D + V - 1) / V;
    if (p.T == 1) {
        const long long blocks = (nvec * p.B + 255) / 256;
        if (blocks > kMaxGroups) return fail(PCRL_E_ARG, "pcrl_short_conv_fwd: too many workgroups");
        conv_step_kernel<T, V, W><<<dim3((unsigned)blocks), 256, 0, s>>>(p);
        PCRL_CHECK_LAUNCH("conv_step_kernel");
        return PCRL_OK;
    }
    p.nrun = (p.T + kRun - 1) / kRun;
    const long long blocks = (nvec * p.B * (p.nrun + 1) + 255) / 256;
    if (blocks > kMaxGroups) return fail(PCRL_E_ARG, "pcrl_short_conv_fwd: too many workgroups");
    conv_fwd_kernel<T, V, W><<<dim3((unsigned)blocks), 256, 0, s>>>(p);
    PCRL_CHECK_LAUNCH("conv_fwd_kernel");
    return PCRL_OK;
}
// Long runs read less halo, short ones fill the chip: the longest of 32, 16, 8 steps with two waves for every SIMD.  Four walkers of 64 channel
// vectors a workgroup, about four workgroups per CU, which leave one part of the sums each.
static void conv_bwd_plan(const pcrl_conv_desc* d, int& run, int& nrun, int& parts) {
    const int V = kConvV;
    const long long cols = (d->D + 64 * V - 1) / (64 * V);
    run = 32;
    while (run > 8 && cols * d->B * ((d->T + run - 1) / run) < 8LL * num_cus()) run >>= 1;
    nrun = (d->T + run - 1) / run;
    const long long lines = (long long)d->B * nrun, want = 4LL * num_cus() / cols;
    long long n = (lines + 3) / 4;
    if (n > want) n = want;
    parts = n < 1 ? 1 : (int)n;
}
template <typename T, int V, int W>
static int conv_bwd(ConvParams& p, float* dweight, float* dbias, hipStream_t s) {
    const size_t lds = sizeof(float) * 4 * (W + 1) * 64 * V;
    const unsigned cols = (unsigned)((p.D + 64 * V - 1) / (64 * V));
    conv_bwd_kernel<T, V, W><<<dim3(cols, (unsigned)p.parts), 256, lds, s>>>(p);
    PCRL_CHECK_LAUNCH("conv_bwd_kernel");
    conv_finish_kernel<<<dim3((unsigned)((p.D + 63) / 64), (unsigned)(W + 1)), 1024, 0, s>>>(p.part, p.parts, W, p.D, dweight, dbias);
    PCRL_CHECK_LAUNCH("conv_finish_kernel");
    return PCRL_OK;
}

}  // namespace pcrl

using namespace pcrl;

#define PCRL_CONV_W(CALL, T, V)                                        \
    switch (d->W) {                                                    \
        case 1: return CALL<T, V, 1> PCRL_CONV_ARGS;                   \
        case 2: return CALL<T, V, 2> PCRL_CONV_ARGS;                   \
        case 3: return CALL<T, V, 3> PCRL_CONV_ARGS;                   \
        default: return CALL<T, V, 4> PCRL_CONV_ARGS;                  \
    }

extern "C" int pcrl_short_conv_fwd(const pcrl_conv_desc* d, void* y, void* last_state, void* stream) {
    if (int rc = conv_check(d, "pcrl_short_conv_fwd")) return rc;
    if (!y) return fail(PCRL_E_ARG, "pcrl_short_conv_fwd: null output");
    if (overlap(last_state, d->state, (size_t)d->B * (d->W - 1) * d->D * elem_bytes(d->dtype), d->T > 1))
        return fail(PCRL_E_ARG, "pcrl_short_conv_fwd: last_state overlaps state (T = %d; a single step may update it in place)", d->T);
    ConvParams p;
    conv_fill(p, d);
    p.y = y, p.last = last_state;
    const void* extra[2] = {y, last_state};
    p.vec = conv_vec(d, kConvV, extra, 2);
    hipStream_t s = (hipStream_t)stream;
#define PCRL_CONV_ARGS (p, s)
    if (d->dtype == PCRL_DT_F32) { PCRL_CONV_W(conv_fwd, float, kConvV) }
    if (d->dtype == PCRL_DT_BF16) { PCRL_CONV_W(conv_fwd, __bf16, kConvV) }
    PCRL_CONV_W(conv_fwd, _Float16, kConvV)
#undef PCRL_CONV_ARGS
}

extern "C" int pcrl_short_conv_bwd_workspace_bytes(const pcrl_conv_desc* d, size_t* bytes) {
    if (int rc = conv_check(d, "pcrl_short_conv_bwd_workspace_bytes")) return rc;
    if (!bytes) return fail(PCRL_E_ARG, "pcrl_short_conv_bwd_workspace_bytes: null output");
    int run, nrun, parts;
    conv_bwd_plan(d, run, nrun, parts);
    *bytes = sizeof(float) * (size_t)parts * (d->W + 1) * d->D;
    return PCRL_OK;
}

extern "C" int pcrl_short_conv_bwd(const pcrl_conv_desc* d, const void* dy, int64_t dy_sb, int64_t dy_st, const void* dlast, void* dx, float* dweight,
                                   float* dbias, void* dstate, void* workspace, size_t workspace_bytes, void* stream) {
    size_t need = 0;
    if (int rc = pcrl_short_conv_bwd_workspace_bytes(d, &need)) return rc;
    if (!dy || !dx || !dweight) return fail(PCRL_E_ARG, "pcrl_short_conv_bwd: null gradient or output");
    if (!workspace || workspace_bytes < need) return fail(PCRL_E_WORKSPACE, "pcrl_short_conv_bwd: workspace %zu < %zu", workspace_bytes, need);
    ConvParams p;
    conv_fill(p, d);
    conv_bwd_plan(d, p.run, p.nrun, p.parts);
    p.dy = dy, p.dy_sb = dy_sb, p.dy_st = dy_st, p.dlast = dlast, p.dx = dx, p.dstate = dstate, p.part = (float*)workspace;
    const int V = kConvV;
    const void* extra[4] = {dy, dlast, dx, dstate};
    p.vec = conv_vec(d, V, extra, 4) && dy_sb % V == 0 && dy_st % V == 0;
    hipStream_t s = (hipStream_t)stream;
#define PCRL_CONV_ARGS (p, dweight, dbias, s)
    if (d->dtype == PCRL_DT_F32) { PCRL_CONV_W(conv_bwd, float, kConvV) }
    if (d->dtype == PCRL_DT_BF16) { PCRL_CONV_W(conv_bwd, __bf16, kConvV) }
    PCRL_CONV_W(conv_bwd, _Float16, kConvV)
#undef PCRL_CONV_ARGS
}
