// Selective state space scan, backward (ssm_common.h: the split; include/pcrl.h: the formulas).
//
//   g_t = C_t ds_t + a_{t+1} g_{t+1}      (a_{t+1} := 0 where step t + 1 begins a new sequence; behind the last step: dlast)
//   dC_t = sum_d ds_t h_t    dB_t = sum_d g_t dt_t u_t
//   du_t = dt_t sum_n g_t B_t + D ds_t    ddt_t = u_t sum_n g_t B_t + sum_n A w_t    dA = sum_t dt_t w_t    with w_t = g_t a_t h_{t-1}
// Tiles are walked from the last to the first.  The states inside a tile are formed again from the state in front of it (left by the forward,
// 4 N / 16 bytes per element: reading it costs less than a second walk from further back), kept in registers with the decays, and met by g on
// the way back.  dB and dC are sums over channels: 16 steps x 4 states of lane values per wave.  Two steps' values are folded into one register
// as soon as both exist (each lane keeps one and sends the other: 3 instructions for 2 values instead of 6 for each value's own tree), left per
// channel block, and added up in a fixed order by a second launch.
#include "ssm_common.h"

namespace pcrl {

// lo / hi: two values per lane -> one: lanes with the level's bit of their row position clear get lo + partner's lo, the others hi + partner's
// hi.  Partners: position ^ 7 (half-row mirror; first, because it mixes the low bits), ^ 2, ^ 1, ^ 8: after the four levels every position of the
// row is in the sum once.  Levels 0 to 3 settle bits 2, 1, 0, 3 of the position.
template <int LEVEL>
__device__ __forceinline__ float fold(float lo, float hi, int r) {
    constexpr int bit = LEVEL == 0 ? 4 : LEVEL == 1 ? 2 : LEVEL == 2 ? 1 : 8;
    const bool up = (r & bit) != 0;
    const float keep = up ? hi : lo, send = up ? lo : hi;
    return keep + dpp_f<LEVEL == 0 ? 0x141 : LEVEL == 1 ? 0x4E : LEVEL == 2 ? 0xB1 : 0x128>(send);
}
// The step whose value a lane at row position r is left with: bits 0 and 2 change places.
__device__ __forceinline__ int folded_step(int r) { return (r & 10) | ((r & 1) << 2) | ((r >> 2) & 1); }
// Binary counter of folds: step t = 15 - K arrives; `held` keeps the upper half of each unfinished pair.  After K = 15 each lane holds in
// held[3] its row's sum of the value of step folded_step(r).
template <int K>
__device__ __forceinline__ void fold_step(float v, float (&held)[4], int r) {
    constexpr int t = 15 - K;
    if constexpr ((t & 1) != 0) { held[0] = v; }
    else {
        const float f0 = fold<0>(v, held[0], r);
        if constexpr ((t & 2) != 0) { held[1] = f0; }
        else {
            const float f1 = fold<1>(f0, held[1], r);
            if constexpr ((t & 4) != 0) { held[2] = f1; }
            else {
                const float f2 = fold<2>(f1, held[2], r);
                held[3] = (t & 8) != 0 ? f2 : fold<3>(f2, held[3], r);
            }
        }
    }
}
__device__ __forceinline__ float add_swapped32(float a, float b) {       // lower half: a's two halves added, upper half: b's
    auto x = __builtin_amdgcn_permlane32_swap(f2u(a), f2u(b), false, false);
    return u2f(x[0]) + u2f(x[1]);
}
__device__ __forceinline__ float add_swapped16(float a, float b) {       // even rows: a's row pair added, odd rows: b's
    auto x = __builtin_amdgcn_permlane16_swap(f2u(a), f2u(b), false, false);
    return u2f(x[0]) + u2f(x[1]);
}

template <typename T, int CPW, bool SUMMARY>
__global__ __launch_bounds__(512) void ssm_bwd_kernel(const SsmParams p) {
    constexpr int NS = CPW / 16, V = CPW / 16, ROWS = 64 / CPW;
    extern __shared__ float lds[];
    const int groups = p.S * ROWS;                      // partial sums over the states of one (step, channel)
    float* s_dt = lds;                                  // [16][CPW]
    float* s_du = s_dt + kTile * CPW;
    float* s_ds = s_du + kTile * CPW;
    float* s_gb = s_ds + kTile * CPW;                   // [groups][16][CPW]: sum_n g B
    float* s_aw = s_gb + groups * kTile * CPW;          // ... sum_n A w
    float* s_y = s_aw + groups * kTile * CPW;           // ... sum_n C h (only with a gate)
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 15;
    int blk, chunk, b0;
    ssm_where(p, blk, chunk, b0);
    if (SUMMARY && chunk == 0) return;                  // nobody ends at the first chunk's summary
    const int g = blk / p.nblk, c_first = (blk - g * p.nblk) * CPW;
    const int tile0 = chunk * p.chunk_tiles, tile1 = tile0 + p.chunk_tiles < p.ntile ? tile0 + p.chunk_tiles : p.ntile;

    const bool item = tid < 256;
    const int row = (tid & 255) / 16, c0 = ((tid & 255) % 16) * V;
    const int left = p.Dg - c_first - c0, nv = item ? (left < V ? left : V) : 0;
    const int d0 = g * p.Dg + c_first + c0;
    float bias[V], skip[V], d_skip[V], d_bias[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bias[i] = i < nv && p.dt_bias ? p.dt_bias[d0 + i] : 0.0f;
        skip[i] = i < nv && p.Dskip ? p.Dskip[d0 + i] : 0.0f;
        d_skip[i] = d_bias[i] = 0.0f;
    }
    const int ch = lane % CPW, n0 = wave * 4 + (lane / CPW) * NS;
    const int dch = g * p.Dg + c_first + ch;
    const bool has = c_first + ch < p.Dg, walks = wave < p.S;
    float A[NS], A2[NS], dA[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        A[j] = walks && has && n0 + j < p.N ? p.A[(long long)dch * p.N + n0 + j] : 0.0f;
        A2[j] = A[j] * kLog2e;
        dA[j] = 0.0f;
    }

    for (int b = b0; b < p.B; b += p.b_step) {
        const int len = ssm_length(p, b);
        const T* pu = (const T*)p.u + b * p.u_sb + d0;
        const T* pd = (const T*)p.dt + b * p.dt_sb + d0;
        const T* pz = p.z ? (const T*)p.z + b * p.z_sb + d0 : nullptr;
        const T* pg = (const T*)p.dy + b * p.dy_sb + d0;
        const T* pB = (const T*)p.Bm + b * p.b_sb + g * p.b_sg;
        const T* pC = (const T*)p.Cm + b * p.c_sb + g * p.c_sg;
        const uint8_t* ps = p.starts ? p.starts + b * p.starts_sb : nullptr;
        const long long orow = (long long)b * p.T;      // dense outputs
        float gc[NS];                                   // what the steps behind add to g of this one
#pragma unroll
        for (int j = 0; j < NS; ++j)
            gc[j] = !SUMMARY && walks && has && n0 + j < p.N && p.dlast ? p.dlast[((long long)b * p.D + dch) * p.N + n0 + j] : 0.0f;
        if (!SUMMARY && walks && has) {
            for (int c = p.nchunk - 1; c > chunk; --c)
#pragma unroll
                for (int j = 0; j < NS; ++j)
                    if (n0 + j < p.N) {
                        const long long at = (((long long)b * p.nchunk + c) * p.N + n0 + j) * p.D + dch;
                        const float P = p.sum_p[at], s = p.sum_s[at];
                        gc[j] = P == 0.0f ? s : __builtin_fmaf(P, gc[j], s);
                    }
        }
        float dt_sum = 0.0f;
        bool cut = false;

        RawVec<T, V> nu, nd, nz, ng;
        T nB[NS], nC[NS];
        float nh[NS];
        unsigned char nst;
        auto fetch = [&](int tile) {
            const int t = tile * kTile + row, n = t < len ? nv : 0;
            if (!SUMMARY) nu = raw_load<T, V>(pu + t * p.u_st, n, p.vec);
            nd = raw_load<T, V>(pd + t * p.dt_st, n, p.vec);
            if (pz) nz = raw_load<T, V>(pz + t * p.z_st, n, p.vec);
            ng = raw_load<T, V>(pg + t * p.dy_st, n, p.vec);
            const int tl = tile * kTile + r;
            const bool on = walks && tl < len;
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                if (!SUMMARY) nB[j] = on && n0 + j < p.N ? pB[tl * p.b_st + n0 + j] : (T)0.0f;
                nC[j] = on && n0 + j < p.N ? pC[tl * p.c_st + n0 + j] : (T)0.0f;
                if (!SUMMARY) nh[j] = walks && has && n0 + j < p.N ? p.saved[(((long long)b * p.ntile + tile) * p.N + n0 + j) * p.D + dch] : 0.0f;
            }
            nst = ps && tl < len ? ps[tl] : (unsigned char)0;
        };
        const int live = (len + kTile - 1) / kTile, end = tile1 < live ? tile1 : live;
        if (!SUMMARY) {                                 // steps behind the length: zeros
            float none[V];
#pragma unroll
            for (int i = 0; i < V; ++i) none[i] = 0.0f;
            for (int tile = tile0 > live ? tile0 : live; tile < tile1; ++tile) {
                const int t = tile * kTile + row, n = t < p.T ? nv : 0;
                raw_store<T, V>((T*)p.du + (orow + t) * p.D + d0, none, n, p.vec);
                raw_store<T, V>((T*)p.ddt + (orow + t) * p.D + d0, none, n, p.vec);
                if (pz) raw_store<T, V>((T*)p.dz + (orow + t) * p.D + d0, none, n, p.vec);
            }
        }
        if (tile0 < end) fetch(end - 1);
        for (int tile = end - 1; tile >= tile0; --tile) {
            const int t0 = tile * kTile;
            const bool here = t0 + row < len;
            float u[V], z[V], gy[V], dt[V], slope[V], ds[V], sig[V], Bv[NS], Cv[NS], h0[NS];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                u[i] = !SUMMARY ? (float)nu.v[i] : 0.0f;
                z[i] = pz ? (float)nz.v[i] : 0.0f;
                gy[i] = (float)ng.v[i];
                const float raw = (float)nd.v[i] + bias[i];
                slope[i] = 1.0f;
                dt[i] = p.softplus ? softplus_(raw, slope[i]) : raw;
                dt[i] = here ? dt[i] : 0.0f;
                sig[i] = pz ? sigmoidf_(z[i]) : 0.0f;
                ds[i] = pz ? gy[i] * (z[i] * sig[i]) : gy[i];
            }
            if (item) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    s_dt[row * CPW + c0 + i] = dt[i];
                    if (!SUMMARY) s_du[row * CPW + c0 + i] = dt[i] * u[i];
                    s_ds[row * CPW + c0 + i] = ds[i];
                }
            }
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                Bv[j] = !SUMMARY ? (float)nB[j] : 0.0f;
                Cv[j] = (float)nC[j];
                h0[j] = !SUMMARY ? nh[j] : 0.0f;
            }
            const unsigned starts = ssm_start_bits(nst);
            if (tile > tile0) fetch(tile - 1);
            __syncthreads();
            if (walks) {
                const int at = (wave * ROWS + lane / CPW) * (kTile * CPW) + ch;
                auto walk = [&](auto with_starts) {
                    constexpr bool WS = decltype(with_starts)::value;
                    if constexpr (SUMMARY) {
                        static_for<kTile>([&](auto ki) {
                            constexpr int t = 15 - decltype(ki)::value;
                            const float dt_ = s_dt[t * CPW + ch], ds_ = s_ds[t * CPW + ch];
                            const bool fresh = WS && ((starts >> t) & 1u);
#pragma unroll
                            for (int j = 0; j < NS; ++j) {
                                const float gt = __builtin_fmaf(row_bcast<t>(Cv[j]), ds_, gc[j]);
                                const float next = gt * __builtin_amdgcn_exp2f(dt_ * A2[j]);
                                gc[j] = fresh ? 0.0f : next;
                            }
                            dt_sum += dt_;
                        });
                    } else {
                        float a[kTile][NS], h[kTile][NS];
                        static_for<kTile>([&](auto ti) {
                            constexpr int t = decltype(ti)::value;
                            const float dt_ = s_dt[t * CPW + ch], du_ = s_du[t * CPW + ch];
                            const bool fresh = WS && ((starts >> t) & 1u);
                            float acc = 0.0f;
#pragma unroll
                            for (int j = 0; j < NS; ++j) {
                                const float x = du_ * row_bcast<t>(Bv[j]), e = __builtin_amdgcn_exp2f(dt_ * A2[j]);
                                const float hn = __builtin_fmaf(e, t == 0 ? h0[j] : h[t == 0 ? 0 : t - 1][j], x);
                                a[t][j] = fresh ? 0.0f : e;
                                h[t][j] = fresh ? x : hn;
                                acc = j == 0 ? h[t][j] * row_bcast<t>(Cv[j]) : __builtin_fmaf(row_bcast<t>(Cv[j]), h[t][j], acc);
                            }
                            if (p.z) s_y[at + t * CPW] = acc;
                        });
                        float hb[NS][4], hc[NS][4];
                        static_for<kTile>([&](auto ki) {
                            constexpr int K = decltype(ki)::value, t = 15 - K;
                            const float dt_ = s_dt[t * CPW + ch], du_ = s_du[t * CPW + ch], ds_ = s_ds[t * CPW + ch];
                            const bool fresh = WS && ((starts >> t) & 1u);
                            float gb = 0.0f, aw = 0.0f;
#pragma unroll
                            for (int j = 0; j < NS; ++j) {
                                const float gt = __builtin_fmaf(row_bcast<t>(Cv[j]), ds_, gc[j]);
                                gb = j == 0 ? gt * row_bcast<t>(Bv[j]) : __builtin_fmaf(row_bcast<t>(Bv[j]), gt, gb);
                                const float gd = gt * a[t][j];
                                float w = gd * (t == 0 ? h0[j] : h[t == 0 ? 0 : t - 1][j]);
                                if (WS) w = fresh ? 0.0f : w;
                                aw = j == 0 ? w * A[j] : __builtin_fmaf(w, A[j], aw);
                                dA[j] = __builtin_fmaf(w, dt_, dA[j]);
                                gc[j] = gd;
                                fold_step<K>(gt * du_, hb[j], r);
                                fold_step<K>(ds_ * h[t][j], hc[j], r);
                            }
                            s_gb[at + t * CPW] = gb;
                            s_aw[at + t * CPW] = aw;
                        });
                        // a lane of a row: one step.  CPW = 64: the four rows hold parts of the sums of 4 states -> one state per row;
                        // CPW = 32: two row pairs with 2 states each -> likewise; CPW = 16: a row is a state already.
                        float vb, vc;
                        if constexpr (CPW == 64) {
                            vb = add_swapped16(add_swapped32(hb[0][3], hb[2][3]), add_swapped32(hb[1][3], hb[3][3]));
                            vc = add_swapped16(add_swapped32(hc[0][3], hc[2][3]), add_swapped32(hc[1][3], hc[3][3]));
                        } else if constexpr (CPW == 32) {
                            vb = add_swapped16(hb[0][3], hb[1][3]);
                            vc = add_swapped16(hc[0][3], hc[1][3]);
                        } else {
                            vb = hb[0][3], vc = hc[0][3];
                        }
                        const int n = wave * 4 + (lane >> 4), ts = t0 + folded_step(r);
                        if (n < p.N && ts < len) {
                            const long long o = (((long long)blk * p.B + b) * p.T + ts) * p.N + n;
                            p.part_b[o] = vb;
                            p.part_c[o] = vc;
                        }
                    }
                };
                if (starts) { walk(std::true_type{}); cut = true; }
                else walk(std::false_type{});
            }
            __syncthreads();
            if (!SUMMARY && item) {
                float gb[V], aw[V], ys[V], o_u[V], o_dt[V], o_z[V];
#pragma unroll
                for (int i = 0; i < V; ++i) gb[i] = aw[i] = ys[i] = 0.0f;
                for (int s = 0; s < groups; ++s)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const int at = s * (kTile * CPW) + row * CPW + c0 + i;
                        gb[i] += s_gb[at];
                        aw[i] += s_aw[at];
                        if (pz) ys[i] += s_y[at];
                    }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    o_u[i] = __builtin_fmaf(dt[i], gb[i], skip[i] * ds[i]);
                    o_dt[i] = here ? __builtin_fmaf(u[i], gb[i], aw[i]) * slope[i] : 0.0f;
                    if (!here) o_u[i] = 0.0f;
                    const float y = __builtin_fmaf(skip[i], u[i], ys[i]);
                    o_z[i] = gy[i] * y * (sig[i] + z[i] * sig[i] * (1.0f - sig[i]));
                    d_skip[i] = __builtin_fmaf(ds[i], u[i], d_skip[i]);
                    d_bias[i] += o_dt[i];
                }
                const int n = t0 + row < p.T ? nv : 0;
                raw_store<T, V>((T*)p.du + (orow + t0 + row) * p.D + d0, o_u, n, p.vec);
                raw_store<T, V>((T*)p.ddt + (orow + t0 + row) * p.D + d0, o_dt, n, p.vec);
                if (pz) raw_store<T, V>((T*)p.dz + (orow + t0 + row) * p.D + d0, o_z, n, p.vec);
            }
        }
        if (walks && has) {
#pragma unroll
            for (int j = 0; j < NS; ++j)
                if (n0 + j < p.N) {
                    if (SUMMARY) {
                        const long long at = (((long long)b * p.nchunk + chunk) * p.N + n0 + j) * p.D + dch;
                        p.sum_p[at] = cut ? 0.0f : __builtin_amdgcn_exp2f(dt_sum * A2[j]);
                        p.sum_s[at] = gc[j];
                    } else if (chunk == 0 && p.dstate) {
                        p.dstate[((long long)b * p.D + dch) * p.N + n0 + j] = gc[j];
                    }
                }
        }
    }
    if (SUMMARY) return;
    // this workgroup's part of dA, dD, ddt_bias
    const long long part = (long long)b0 * p.nchunk + chunk;
    if (walks && has) {
#pragma unroll
        for (int j = 0; j < NS; ++j)
            if (n0 + j < p.N) p.part_a[(part * p.N + n0 + j) * p.D + dch] = dA[j];
    }
    __syncthreads();
    if (item) {
#pragma unroll
        for (int i = 0; i < V; ++i) { s_dt[row * CPW + c0 + i] = d_skip[i]; s_du[row * CPW + c0 + i] = d_bias[i]; }
    }
    __syncthreads();
    if (tid < CPW && c_first + tid < p.Dg) {
        float x = 0.0f, y = 0.0f;
#pragma unroll
        for (int t = 0; t < kTile; ++t) { x += s_dt[t * CPW + tid]; y += s_du[t * CPW + tid]; }
        p.part_d[part * p.D + g * p.Dg + c_first + tid] = x;
        p.part_bias[part * p.D + g * p.Dg + c_first + tid] = y;
    }
}

// Adds the parts up in a fixed order.  Workgroups 0 ... n_par - 1: 64 channels of one row of (dA: N rows, dD, ddt_bias), 16 threads a channel
// over the parts; the others: 1024 elements of dB or dC over the channel blocks of their group.
struct SsmFinishParams {
    int B, T, D, N, G, nblk, parts, n_par, dblk;
    const float *part_a, *part_d, *part_bias, *part_b, *part_c;
    float *dA, *dD, *ddt_bias;
    void *dB, *dC;
    const int* lengths;
};
template <typename T>
__global__ __launch_bounds__(1024) void ssm_finish_kernel(const SsmFinishParams p) {
    __shared__ float s_sum[16][64];
    if ((int)blockIdx.x < p.n_par) {
        const int rowi = blockIdx.x / p.dblk, d = (blockIdx.x - rowi * p.dblk) * 64 + (threadIdx.x & 63), k = threadIdx.x >> 6;
        const float* src = rowi < p.N ? p.part_a + (long long)rowi * p.D : rowi == p.N ? p.part_d : p.part_bias;
        const long long step = rowi < p.N ? (long long)p.N * p.D : p.D;
        float sum = 0.0f;
        if (d < p.D) {
#pragma unroll 8
            for (int i = k; i < p.parts; i += 16) sum += src[i * step + d];
        }
        s_sum[k][threadIdx.x & 63] = sum;
        __syncthreads();
        if (threadIdx.x < 64 && d < p.D) {
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) t += s_sum[i][threadIdx.x];
            if (rowi < p.N) p.dA[(long long)d * p.N + rowi] = t;
            else if (rowi == p.N) { if (p.dD) p.dD[d] = t; }
            else if (p.ddt_bias) p.ddt_bias[d] = t;
        }
        return;
    }
    // element (b, t, g, n) of dB / dC
    const long long per = (long long)p.B * p.T * p.G * p.N, i = (long long)(blockIdx.x - p.n_par) * 1024 + threadIdx.x;
    if (i >= 2 * per) return;
    const bool second = i >= per;
    const long long e = second ? i - per : i;
    const int n = (int)(e % p.N);
    const long long q = e / p.N;
    const int g = (int)(q % p.G);
    const long long bt = q / p.G;
    const int b = (int)(bt / p.T), t = (int)(bt - (long long)b * p.T);
    float sum = 0.0f;
    if (!p.lengths || t < p.lengths[b]) {
        const float* src = (second ? p.part_c : p.part_b) + ((long long)g * p.nblk * p.B * p.T + bt) * p.N + n;
        const long long step = (long long)p.B * p.T * p.N;
#pragma unroll 8
        for (int k = 0; k < p.nblk; ++k) sum += src[k * step];
    }
    ((T*)(second ? p.dC : p.dB))[e] = (T)sum;
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------
// Batch rows that share a workgroup (their dA sums stay in registers): as many as leave about four workgroups per CU.
static int bwd_b_step(const pcrl_ssm_desc* d, const SsmPlan& plan) {
    if (plan.nchunk > 1) return d->B;
    const long long want = 4LL * num_cus() / ((long long)d->G * plan.nblk);
    return want < 1 ? 1 : want < d->B ? (int)want : d->B;
}

struct BwdLayout { size_t b, c, a, dskip, bias, p, s, total; };
static BwdLayout bwd_layout(const pcrl_ssm_desc* d, const SsmPlan& plan) {
    BwdLayout o{};
    size_t at = 0;
    auto take = [&](size_t n) { const size_t was = at; at += (n + 63) & ~(size_t)63; return was; };
    const size_t parts = (size_t)bwd_b_step(d, plan) * plan.nchunk, bc = (size_t)d->G * plan.nblk * d->B * d->T * d->N;
    o.b = take(bc), o.c = take(bc);
    o.a = take(parts * d->N * d->D), o.dskip = take(parts * d->D), o.bias = take(parts * d->D);
    const size_t sum = plan.nchunk > 1 ? (size_t)d->B * plan.nchunk * d->N * d->D : 0;
    o.p = take(sum), o.s = take(sum);
    o.total = at * sizeof(float);
    return o;
}
size_t ssm_bwd_workspace(const pcrl_ssm_desc* d) { return bwd_layout(d, ssm_plan(d)).total; }

template <typename T, int CPW>
static int launch_bwd(const SsmParams& p, hipStream_t s) {
    const int waves = ssm_waves(p.N), rows = 64 / CPW;
    const size_t lds = sizeof(float) * kTile * CPW * (3 + (size_t)(p.z ? 3 : 2) * p.S * rows);
    const dim3 grid((unsigned)(p.G * p.nblk) * p.nchunk * (p.b_step < p.B ? p.b_step : p.B));
    if (p.nchunk > 1) {
        ssm_bwd_kernel<T, CPW, true><<<grid, 64 * waves, sizeof(float) * kTile * CPW * 3, s>>>(p);
        PCRL_CHECK_LAUNCH("ssm_bwd_kernel (summary)");
    }
    if (int rc = ensure_dynamic_lds((const void*)ssm_bwd_kernel<T, CPW, false>, lds)) return rc;
    ssm_bwd_kernel<T, CPW, false><<<grid, 64 * waves, lds, s>>>(p);
    PCRL_CHECK_LAUNCH("ssm_bwd_kernel");
    return PCRL_OK;
}
template <typename T>
static int launch_bwd_t(const SsmParams& p, int cpw, const SsmFinishParams& f, hipStream_t s) {
    if (int rc = cpw == 64 ? launch_bwd<T, 64>(p, s) : cpw == 32 ? launch_bwd<T, 32>(p, s) : launch_bwd<T, 16>(p, s)) return rc;
    const long long elems = 2LL * p.B * p.T * p.G * p.N;
    ssm_finish_kernel<T><<<dim3((unsigned)(f.n_par + (elems + 1023) / 1024)), 1024, 0, s>>>(f);
    PCRL_CHECK_LAUNCH("ssm_finish_kernel");
    return PCRL_OK;
}

}  // namespace pcrl

using namespace pcrl;

extern "C" int pcrl_ssm_scan_bwd(const pcrl_ssm_desc* d, const float* saved, const void* dy, int64_t dy_sb, int64_t dy_st, const float* dlast,
                                 const pcrl_ssm_grads* g, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = ssm_check(d, "pcrl_ssm_scan_bwd")) return rc;
    if (!saved || !dy || !g || !g->du || !g->ddt || !g->dB || !g->dC || !g->dA || (d->z && !g->dz))
        return fail(PCRL_E_ARG, "pcrl_ssm_scan_bwd: null saved state, gradient or output");
    const SsmPlan plan = ssm_plan(d);
    const BwdLayout at = bwd_layout(d, plan);
    if (!workspace || workspace_bytes < at.total) return fail(PCRL_E_WORKSPACE, "pcrl_ssm_scan_bwd: workspace %zu < %zu", workspace_bytes, at.total);
    const long long elems = 2LL * d->B * d->T * d->G * d->N;
    if ((long long)d->G * plan.nblk * plan.nchunk * d->B > 0x7FFFFFFFLL || elems / 1024 > 0x3FFFFFFFLL) return fail(PCRL_E_ARG, "pcrl_ssm_scan_bwd: too many workgroups");
    float* w = (float*)workspace;
    SsmParams p;
    ssm_fill(p, d);
    p.nblk = plan.nblk, p.nchunk = plan.nchunk, p.chunk_tiles = plan.chunk_tiles;
    p.b_step = bwd_b_step(d, plan), p.parts = p.b_step * plan.nchunk;
    p.saved = const_cast<float*>(saved), p.dy = dy, p.dy_sb = dy_sb, p.dy_st = dy_st, p.dlast = dlast;
    p.du = g->du, p.ddt = g->ddt, p.dz = g->dz, p.dstate = g->dstate;
    p.part_b = w + at.b, p.part_c = w + at.c, p.part_a = w + at.a, p.part_d = w + at.dskip, p.part_bias = w + at.bias;
    p.sum_p = w + at.p, p.sum_s = w + at.s;
    const void* extra[4] = {dy, g->du, g->ddt, g->dz};
    const long long dense[2] = {(long long)d->T * d->D, d->D};
    const long long strides[8] = {dy_sb, dy_st, dense[0], dense[1], dense[0], dense[1], dense[0], dense[1]};
    p.vec = ssm_vec(d, plan.cpw / 16, extra, strides, 4);
    SsmFinishParams f{};
    f.B = d->B, f.T = d->T, f.D = d->D, f.N = d->N, f.G = d->G, f.nblk = plan.nblk, f.parts = p.parts;
    f.dblk = cdiv(d->D, 64), f.n_par = (d->N + 2) * f.dblk;
    f.part_a = p.part_a, f.part_d = p.part_d, f.part_bias = p.part_bias, f.part_b = p.part_b, f.part_c = p.part_c;
    f.dA = g->dA, f.dD = g->dD, f.ddt_bias = g->ddt_bias, f.dB = g->dB, f.dC = g->dC, f.lengths = d->lengths;
    hipStream_t s = (hipStream_t)stream;
    return d->dtype == PCRL_DT_F32 ? launch_bwd_t<float>(p, plan.cpw, f, s) : d->dtype == PCRL_DT_BF16 ? launch_bwd_t<__bf16>(p, plan.cpw, f, s) : launch_bwd_t<_Float16>(p, plan.cpw, f, s);
}
