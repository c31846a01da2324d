// Selective state space scan, forward and single step (ssm_common.h: the split; include/pcrl.h: the formulas).
#include "ssm_common.h"

namespace pcrl {

// SUMMARY: only the states are walked, from zero, and the chunk's summary (product of the decays, end state) is left; otherwise the chunk
// starts from the combined summaries of the chunks in front of it and y is written.
template <typename T, int CPW, bool SUMMARY>
__global__ __launch_bounds__(512) void ssm_fwd_kernel(const SsmParams p) {
    constexpr int NS = CPW / 16, V = CPW / 16, ROWS = 64 / CPW;       // states per lane, channels per thread, state rows per wave
    extern __shared__ float lds[];
    float* s_dt = lds;                                  // [16][CPW]
    float* s_du = lds + kTile * CPW;                    // [16][CPW]
    float* s_y = lds + 2 * kTile * CPW;                 // [S * ROWS][16][CPW]
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    int blk, chunk, b;
    ssm_where(p, blk, chunk, b);
    if (SUMMARY && chunk == p.nchunk - 1) return;       // nobody starts from the last chunk's summary
    const int g = blk / p.nblk, c_first = (blk - g * p.nblk) * CPW;   // first channel of this block inside its group
    const int len = ssm_length(p, b);
    const int tile0 = chunk * p.chunk_tiles, tile1 = tile0 + p.chunk_tiles < p.ntile ? tile0 + p.chunk_tiles : p.ntile;

    // the thread's item of a tile: step `row`, channels c0 ... c0 + V - 1
    const bool item = tid < 256;
    const int row = (tid & 255) / 16, c0 = ((tid & 255) % 16) * V;
    const int left = p.Dg - c_first - c0, nv = item ? (left < V ? left : V) : 0;
    const int d0 = g * p.Dg + c_first + c0;             // global channel
    float bias[V], skip[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bias[i] = i < nv && p.dt_bias ? p.dt_bias[d0 + i] : 0.0f;
        skip[i] = i < nv && p.Dskip ? p.Dskip[d0 + i] : 0.0f;
    }
    const T* pu = (const T*)p.u + b * p.u_sb + d0;
    const T* pd = (const T*)p.dt + b * p.dt_sb + d0;
    const T* pz = p.z ? (const T*)p.z + b * p.z_sb + d0 : nullptr;
    T* py = (T*)p.y + ((long long)b * p.T) * p.D + d0;

    // the lane's states: channel `ch` of the block, states n0 ... n0 + NS - 1
    const int ch = lane % CPW, n0 = wave * 4 + (lane / CPW) * NS;
    const int dch = g * p.Dg + c_first + ch;
    const bool has = c_first + ch < p.Dg;
    const bool walks = wave < p.S;
    float A2[NS], h[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        const bool on = walks && has && n0 + j < p.N;
        A2[j] = on ? p.A[(long long)dch * p.N + n0 + j] * kLog2e : 0.0f;
        h[j] = !SUMMARY && on && p.state ? p.state[((long long)b * p.D + dch) * p.N + n0 + j] : 0.0f;
    }
    if (!SUMMARY && walks && has) {                     // h = P h + S over the chunks in front
        for (int c = 0; c < chunk; ++c) {
#pragma unroll
            for (int j = 0; j < NS; ++j)
                if (n0 + j < p.N) {
                    const long long at = (((long long)b * p.nchunk + c) * p.N + n0 + j) * p.D + dch;
                    const float P = p.sum_p[at], s = p.sum_s[at];
                    h[j] = P == 0.0f ? s : __builtin_fmaf(P, h[j], s);
                }
        }
    }
    const T* pB = (const T*)p.Bm + b * p.b_sb + g * p.b_sg;
    const T* pC = (const T*)p.Cm + b * p.c_sb + g * p.c_sg;
    const uint8_t* ps = p.starts ? p.starts + b * p.starts_sb : nullptr;
    float dt_sum = 0.0f;
    bool cut = false;                                   // a start inside the chunk: nothing from before reaches its end

    RawVec<T, V> nu, nd, nz;
    T nB[NS], nC[NS];
    unsigned char nst;
    auto fetch = [&](int tile) {
        const int t = tile * kTile + row, n = t < len ? nv : 0;
        nu = raw_load<T, V>(pu + t * p.u_st, n, p.vec);
        nd = raw_load<T, V>(pd + t * p.dt_st, n, p.vec);
        if (!SUMMARY && pz) nz = raw_load<T, V>(pz + t * p.z_st, n, p.vec);
        const int tl = tile * kTile + (lane & 15);
        const bool on = walks && tl < len;
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            nB[j] = on && n0 + j < p.N ? pB[tl * p.b_st + n0 + j] : (T)0.0f;
            if (!SUMMARY) nC[j] = on && n0 + j < p.N ? pC[tl * p.c_st + n0 + j] : (T)0.0f;
        }
        nst = ps && tl < len ? ps[tl] : (unsigned char)0;
    };
    const int live = (len + kTile - 1) / kTile, end = tile1 < live ? tile1 : live;      // tiles with a step in them
    if (tile0 < end) fetch(tile0);
    for (int tile = tile0; tile < end; ++tile) {
        const int t0 = tile * kTile;
        float u[V], z[V], Bv[NS], Cv[NS];
        const bool here = t0 + row < len;
        {
            float dt[V], du[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                u[i] = (float)nu.v[i];
                z[i] = !SUMMARY && pz ? (float)nz.v[i] : 0.0f;
                float slope;
                const float raw = (float)nd.v[i] + bias[i];
                dt[i] = p.softplus ? softplus_(raw, slope) : raw;
                dt[i] = here ? dt[i] : 0.0f;            // a step behind the length changes nothing: decay 1, input 0
                du[i] = dt[i] * u[i];
            }
            if (item) {
#pragma unroll
                for (int i = 0; i < V; ++i) { s_dt[row * CPW + c0 + i] = dt[i]; s_du[row * CPW + c0 + i] = du[i]; }
            }
        }
#pragma unroll
        for (int j = 0; j < NS; ++j) { Bv[j] = (float)nB[j]; Cv[j] = !SUMMARY ? (float)nC[j] : 0.0f; }
        const unsigned starts = ssm_start_bits(nst);
        if (tile + 1 < end) fetch(tile + 1);
        __syncthreads();
        if (walks) {
            if (!SUMMARY && p.saved && has) {
#pragma unroll
                for (int j = 0; j < NS; ++j)
                    if (n0 + j < p.N) p.saved[(((long long)b * p.ntile + tile) * p.N + n0 + j) * p.D + dch] = h[j];
            }
            float* out = s_y + (wave * ROWS + lane / CPW) * (kTile * CPW) + ch;
            auto walk = [&](auto with_starts) {
                static_for<kTile>([&](auto ti) {
                    constexpr int t = decltype(ti)::value;
                    const float dt = s_dt[t * CPW + ch], du = s_du[t * CPW + ch];
                    const bool fresh = decltype(with_starts)::value && ((starts >> t) & 1u);
                    float acc = 0.0f;
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        const float x = du * row_bcast<t>(Bv[j]);
                        const float a = __builtin_amdgcn_exp2f(dt * A2[j]);
                        const float hn = __builtin_fmaf(a, h[j], x);
                        h[j] = fresh ? x : hn;
                        if (!SUMMARY) acc = j == 0 ? h[j] * row_bcast<t>(Cv[j]) : __builtin_fmaf(row_bcast<t>(Cv[j]), h[j], acc);
                    }
                    if (SUMMARY) dt_sum += dt;
                    else out[t * CPW] = acc;
                });
            };
            if (starts) { walk(std::true_type{}); cut = true; }
            else walk(std::false_type{});
        }
        __syncthreads();
        if (!SUMMARY && item) {
            float acc[V];
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = 0.0f;
            for (int s = 0; s < p.S * ROWS; ++s)
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] += s_y[s * (kTile * CPW) + row * CPW + c0 + i];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                acc[i] = __builtin_fmaf(skip[i], u[i], acc[i]);
                if (pz) acc[i] *= z[i] * sigmoidf_(z[i]);
                acc[i] = here ? acc[i] : 0.0f;
            }
            raw_store<T, V>(py + (long long)(t0 + row) * p.D, acc, t0 + row < p.T ? nv : 0, p.vec);
        }
    }
    if (!SUMMARY) {                                     // steps behind the length: zeros
        float none[V];
#pragma unroll
        for (int i = 0; i < V; ++i) none[i] = 0.0f;
        for (int tile = tile0 > live ? tile0 : live; tile < tile1; ++tile)
            raw_store<T, V>(py + (long long)(tile * kTile + row) * p.D, none, tile * kTile + row < p.T ? nv : 0, p.vec);
    }
    if (walks && has) {
#pragma unroll
        for (int j = 0; j < NS; ++j)
            if (n0 + j < p.N) {
                if (SUMMARY) {
                    const long long at = (((long long)b * p.nchunk + chunk) * p.N + n0 + j) * p.D + dch;
                    p.sum_p[at] = cut ? 0.0f : __builtin_amdgcn_exp2f(dt_sum * A2[j]);
                    p.sum_s[at] = h[j];
                } else if (p.last && chunk == p.nchunk - 1) {
                    p.last[((long long)b * p.D + dch) * p.N + n0 + j] = h[j];
                }
            }
    }
}

// One step.  The state is 8 N bytes per channel of traffic against a few of everything else, so lanes run along it: LPC lanes per channel, four
// states each (16-byte accesses when N % 4 == 0), the sum over the states inside the group of LPC lanes.
struct SsmStepParams {
    SsmParams s;
    float* state_out;
    int lpc;                           // lanes per channel: 1, 2, 4 or 8
    int vec4;                          // N % 4 == 0 and A and the states aligned: whole 16-byte accesses
};
template <typename T>
__global__ __launch_bounds__(256) void ssm_step_kernel(const SsmStepParams q) {
    const SsmParams& p = q.s;
    const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long pair = idx / q.lpc;
    const int k = (int)(idx - pair * q.lpc) * 4;
    const bool on = pair < (long long)p.B * p.D;
    const int b = on ? (int)(pair / p.D) : 0, d = on ? (int)(pair - (long long)b * p.D) : 0, g = d / p.Dg;
    const int n = on ? (p.N - k < 4 ? p.N - k : 4) : 0;
    const bool vec = q.vec4;
    const float u = on ? (float)((const T*)p.u)[b * p.u_sb + d] : 0.0f;
    float dt = on ? (float)((const T*)p.dt)[b * p.dt_sb + d] + (p.dt_bias ? p.dt_bias[d] : 0.0f) : 0.0f, slope;
    if (p.softplus) dt = softplus_(dt, slope);
    const bool fresh = on && p.starts && p.starts[b * p.starts_sb];
    const RawVec<float, 4> h = raw_load<float, 4>(p.state + pair * p.N + k, fresh ? 0 : n, vec);
    const RawVec<float, 4> A = raw_load<float, 4>(p.A + (long long)d * p.N + k, n, vec);
    const RawVec<T, 4> Bv = raw_load<T, 4>((const T*)p.Bm + b * p.b_sb + g * p.b_sg + k, n, false);
    const RawVec<T, 4> Cv = raw_load<T, 4>((const T*)p.Cm + b * p.c_sb + g * p.c_sg + k, n, false);
    const float du = dt * u;
    float out[4], acc = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float x = du * (float)Bv.v[j];
        out[j] = fresh ? x : __builtin_fmaf(__builtin_amdgcn_exp2f(dt * (A.v[j] * kLog2e)), h.v[j], x);
        acc = j < n ? __builtin_fmaf((float)Cv.v[j], out[j], acc) : acc;
    }
    raw_store<float, 4>(q.state_out + pair * p.N + k, out, n, vec);
    for (int off = q.lpc >> 1; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
    if (on && k == 0) {
        if (p.Dskip) acc = __builtin_fmaf(p.Dskip[d], u, acc);
        if (p.z) {
            const float z = (float)((const T*)p.z)[b * p.z_sb + d];
            acc *= z * sigmoidf_(z);
        }
        ((T*)p.y)[pair] = (T)acc;
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------
int ssm_check(const pcrl_ssm_desc* d, const char* who) {
    if (!d) return fail(PCRL_E_ARG, "%s: null descriptor", who);
    if (d->B < 1 || d->T < 1 || d->D < 1 || d->N < 1 || d->G < 1) return fail(PCRL_E_ARG, "%s: B, T, D, N, G must be positive (%d, %d, %d, %d, %d)", who, d->B, d->T, d->D, d->N, d->G);
    if (d->N > kSsmMaxN) return fail(PCRL_E_ARG, "%s: N = %d states per channel (at most %d)", who, d->N, kSsmMaxN);
    if (d->D % d->G) return fail(PCRL_E_ARG, "%s: %d channels are not shared evenly by %d groups", who, d->D, d->G);
    if (!seq_dtype(d->dtype)) return fail(PCRL_E_ARG, "%s: dtype %d", who, d->dtype);
    if (!d->u || !d->dt || !d->Bm || !d->Cm || !d->A) return fail(PCRL_E_ARG, "%s: null input", who);
    return PCRL_OK;
}

void ssm_fill(SsmParams& p, const pcrl_ssm_desc* d) {
    p = SsmParams{};
    p.B = d->B, p.T = d->T, p.D = d->D, p.N = d->N, p.G = d->G, p.Dg = d->D / d->G;
    p.S = cdiv(d->N, 4);
    p.softplus = d->softplus != 0;
    p.ntile = cdiv(d->T, kTile);
    p.u = d->u, p.dt = d->dt, p.z = d->z, p.Bm = d->Bm, p.Cm = d->Cm;
    p.u_sb = d->u_sb, p.u_st = d->u_st, p.dt_sb = d->dt_sb, p.dt_st = d->dt_st, p.z_sb = d->z_sb, p.z_st = d->z_st;
    p.b_sb = d->b_sb, p.b_st = d->b_st, p.b_sg = d->b_sg, p.c_sb = d->c_sb, p.c_st = d->c_st, p.c_sg = d->c_sg;
    p.A = d->A, p.Dskip = d->D_skip, p.dt_bias = d->dt_bias, p.state = d->state;
    p.starts = d->starts, p.starts_sb = d->starts_sb, p.lengths = d->lengths;
}

// Whole-vector accesses: V channels of every row start at a multiple of V elements.
bool ssm_vec(const pcrl_ssm_desc* d, int V, const void* const* extra, const long long* strides, int n_extra) {
    const size_t bytes = (size_t)V * elem_bytes(d->dtype);
    if ((d->D / d->G) % V) return false;
    const void* ptr[3] = {d->u, d->dt, d->z};
    const long long st[3][2] = {{d->u_sb, d->u_st}, {d->dt_sb, d->dt_st}, {d->z_sb, d->z_st}};
    for (int i = 0; i < 3; ++i) {
        if (!ptr[i]) continue;
        if ((uintptr_t)ptr[i] % bytes || st[i][0] % V || st[i][1] % V) return false;
    }
    for (int i = 0; i < n_extra; ++i) {
        if (!extra[i]) continue;
        if ((uintptr_t)extra[i] % bytes || strides[2 * i] % V || strides[2 * i + 1] % V) return false;
    }
    return true;
}

SsmPlan ssm_plan(const pcrl_ssm_desc* d) {
    const int Dg = d->D / d->G, ntile = cdiv(d->T, kTile);
    const long long cus = num_cus();
    SsmPlan plan{};
    for (int cpw = 64; cpw >= 16; cpw >>= 1) {
        plan.cpw = cpw, plan.nblk = cdiv(Dg, cpw);
        if ((long long)d->B * d->G * plan.nblk >= cus) break;
    }
    const long long blocks = (long long)d->B * d->G * plan.nblk, want = 8 * cus / blocks;
    const int most = ntile / 8 < 1 ? 1 : ntile / 8;
    const int chunks = want < 4 || most < 4 ? 1 : want < most ? (int)want : most;
    plan.chunk_tiles = cdiv(ntile, chunks);
    plan.nchunk = cdiv(ntile, plan.chunk_tiles);
    return plan;
}

template <typename T, int CPW>
static int launch_fwd(SsmParams& p, hipStream_t s) {
    const int waves = ssm_waves(p.N), rows = 64 / CPW;
    const size_t lds = sizeof(float) * kTile * CPW * (2 + (size_t)p.S * rows);
    if (p.nchunk > 1) {
        ssm_fwd_kernel<T, CPW, true><<<dim3((unsigned)(p.G * p.nblk) * p.nchunk * p.B), 64 * waves, sizeof(float) * kTile * CPW * 2, s>>>(p);
        PCRL_CHECK_LAUNCH("ssm_fwd_kernel (summary)");
    }
    ssm_fwd_kernel<T, CPW, false><<<dim3((unsigned)(p.G * p.nblk) * p.nchunk * p.B), 64 * waves, lds, s>>>(p);
    PCRL_CHECK_LAUNCH("ssm_fwd_kernel");
    return PCRL_OK;
}
template <typename T>
static int launch_fwd_t(SsmParams& p, int cpw, hipStream_t s) {
    return cpw == 64 ? launch_fwd<T, 64>(p, s) : cpw == 32 ? launch_fwd<T, 32>(p, s) : launch_fwd<T, 16>(p, s);
}

static size_t fwd_workspace(const pcrl_ssm_desc* d, const SsmPlan& plan) {
    return plan.nchunk > 1 ? sizeof(float) * 2 * (size_t)d->B * plan.nchunk * d->N * d->D : 0;
}
size_t ssm_bwd_workspace(const pcrl_ssm_desc* d);       // ssm_bwd.hip

}  // namespace pcrl

using namespace pcrl;

extern "C" int pcrl_ssm_scan_bytes(const pcrl_ssm_desc* d, size_t* workspace, size_t* saved, size_t* bwd) {
    if (int rc = ssm_check(d, "pcrl_ssm_scan_bytes")) return rc;
    if (workspace) *workspace = fwd_workspace(d, ssm_plan(d));
    if (saved) *saved = sizeof(float) * (size_t)d->B * cdiv(d->T, kTile) * d->N * d->D;
    if (bwd) *bwd = ssm_bwd_workspace(d);
    return PCRL_OK;
}

extern "C" int pcrl_ssm_scan_fwd(const pcrl_ssm_desc* d, void* y, float* last_state, float* saved, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = ssm_check(d, "pcrl_ssm_scan_fwd")) return rc;
    if (!y) return fail(PCRL_E_ARG, "pcrl_ssm_scan_fwd: null output");
    const SsmPlan plan = ssm_plan(d);
    const size_t need = fwd_workspace(d, plan);
    if (need && (!workspace || workspace_bytes < need)) return fail(PCRL_E_WORKSPACE, "pcrl_ssm_scan_fwd: workspace %zu < %zu", workspace_bytes, need);
    if ((long long)d->G * plan.nblk * plan.nchunk * d->B > 0x7FFFFFFFLL) return fail(PCRL_E_ARG, "pcrl_ssm_scan_fwd: too many workgroups");
    SsmParams p;
    ssm_fill(p, d);
    p.nblk = plan.nblk, p.nchunk = plan.nchunk, p.chunk_tiles = plan.chunk_tiles;
    p.y = y, p.last = last_state, p.saved = saved;
    p.sum_p = (float*)workspace, p.sum_s = p.sum_p + (size_t)d->B * plan.nchunk * d->N * d->D;
    const void* extra[1] = {y};
    const long long strides[2] = {(long long)d->T * d->D, d->D};
    p.vec = ssm_vec(d, plan.cpw / 16, extra, strides, 1);
    hipStream_t s = (hipStream_t)stream;
    return d->dtype == PCRL_DT_F32 ? launch_fwd_t<float>(p, plan.cpw, s) : d->dtype == PCRL_DT_BF16 ? launch_fwd_t<__bf16>(p, plan.cpw, s) : launch_fwd_t<_Float16>(p, plan.cpw, s);
}

extern "C" int pcrl_ssm_step(const pcrl_ssm_desc* d, void* y, float* state_out, void* stream) {
    if (int rc = ssm_check(d, "pcrl_ssm_step")) return rc;
    if (d->T != 1) return fail(PCRL_E_ARG, "pcrl_ssm_step: T = %d", d->T);
    if (!y || !state_out || !d->state) return fail(PCRL_E_ARG, "pcrl_ssm_step: null output or state");
    SsmStepParams q;
    ssm_fill(q.s, d);
    q.s.y = y, q.state_out = state_out;
    q.vec4 = (d->N & 3) == 0 && ((uintptr_t)d->state | (uintptr_t)state_out | (uintptr_t)d->A) % 16 == 0;
    q.lpc = d->N <= 4 ? 1 : d->N <= 8 ? 2 : d->N <= 16 ? 4 : 8;
    const long long threads = (long long)d->B * d->D * q.lpc;
    if ((threads + 255) / 256 > 0x7FFFFFFFLL) return fail(PCRL_E_ARG, "pcrl_ssm_step: too many workgroups");
    const dim3 grid((unsigned)((threads + 255) / 256));
    hipStream_t s = (hipStream_t)stream;
    if (d->dtype == PCRL_DT_F32) ssm_step_kernel<float><<<grid, 256, 0, s>>>(q);
    else if (d->dtype == PCRL_DT_BF16) ssm_step_kernel<__bf16><<<grid, 256, 0, s>>>(q);
    else ssm_step_kernel<_Float16><<<grid, 256, 0, s>>>(q);
    PCRL_CHECK_LAUNCH("ssm_step_kernel");
    return PCRL_OK;
}
