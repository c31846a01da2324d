// Selective state space scan, forward and single step (ssm_common.h: the split; include/pcrl.h: the formulas).
//
// The walk is bound by vector instructions: per state and step an exponential, two multiplies and two multiply-adds (its bytes alone would take
// 25 us at 16.8 M elements, N = 16, bf16).  Measured there (4 x 2048 x 2048): 64 us for the chunk summaries and 93 us for the walk, whose 33.3 M
// wave instructions (8 a state and step) are 65 us of every SIMD at 4.3 cycles each; 1 x 16384 x 1024: 62 and 111 us.
#include "ssm_common.h"

namespace pcrl {

// SUMMARY: only the states are walked, from zero, and the chunk's summary (product of the decays, end state) is left; otherwise the chunk
// starts from the combined summaries of the chunks in front of it and y is written.
template <typename T, int RN, int NG, bool VEC, bool SUMMARY>
__global__ __launch_bounds__(256) void ssm_fwd_kernel(const SsmParams) {
    const SsmArgs p = ssm_args();
    constexpr int kWave = 2 * kInTile + (SUMMARY ? 0 : kPartTile);
    __shared__ float lds[4 * kWave];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    float* s_dt = lds + wave * kWave;                   // [channel][step]
    float* s_du = s_dt + kInTile;
    float* s_y = s_du + kInTile;                        // [state row][step][channel]: sum_n C h
    int blk, chunk, b;
    ssm_where(p, blk, chunk, b);
    if (SUMMARY && chunk == p->nchunk - 1) return;       // nobody starts from the last chunk's summary
    const int g = blk / p->nblk, c_first = (blk - g * p->nblk) * 64 + wave * 16;        // first channel of this wave inside its group
    const int left = p->Dg - c_first;                    // channels from there on
    if (left <= 0) return;
    const int len = ssm_length(p, b), d_first = g * p->Dg + c_first;
    const int tile0 = chunk * p->chunk_tiles, tile1 = tile0 + p->chunk_tiles < p->ntile ? tile0 + p->chunk_tiles : p->ntile;

    // loading layout: step `row` of the tile, channels c0 ... c0 + 3 of the wave (clamped to what exists)
    const int row = lane >> 2, c0 = (lane & 3) * 4, nv = left - c0 < 4 ? left - c0 : 4;
    unsigned cc[4];
    float bias[4], skip[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        cc[i] = c0 + i < left ? c0 + i : (VEC ? 0 : left - 1);
        bias[i] = i < nv && p->dt_bias ? p->dt_bias[d_first + c0 + i] : 0.0f;
        skip[i] = i < nv && p->Dskip ? p->Dskip[d_first + c0 + i] : 0.0f;
    }
    const T* pu = (const T*)p->u + b * p->u_sb + d_first;
    const T* pd = (const T*)p->dt + b * p->dt_sb + d_first;
    const T* pz = p->z ? (const T*)p->z + b * p->z_sb + d_first : nullptr;
    T* py = (T*)p->y + (long long)b * p->T * p->D + d_first;

    // walking layout: channel ch of the wave, states n0(k) ... n0(k) + RN - 1 of group k
    const int ch = lane & 15, q = lane >> 4, dch = d_first + ch;
    const bool has = ch < left;
    auto n0 = [&](int k) { return (k * 4 + q) * RN; };
    auto count = [&](int k) { const int n = p->N - n0(k); return has ? (n < RN ? n : RN) : 0; };
    unsigned nn[NG][RN];
    float A2[NG][RN], h[NG][RN];
#pragma unroll
    for (int k = 0; k < NG; ++k) {
        const RawVec<float, RN> a = raw_load<float, RN>(p->A + (long long)dch * p->N + n0(k), count(k), p->vec_n);
        const RawVec<float, RN> s = raw_load<float, RN>(p->state + ((long long)b * p->D + dch) * p->N + n0(k), !SUMMARY && p->state ? count(k) : 0, p->vec_n);
#pragma unroll
        for (int j = 0; j < RN; ++j) {
            A2[k][j] = a.v[j] * kLog2e;
            h[k][j] = s.v[j];
            nn[k][j] = n0(k) + j < p->N ? n0(k) + j : (VEC ? 0 : p->N - 1);
        }
        if (!SUMMARY && chunk > 0) {                    // from the chunks in front
            const long long at = ((long long)b * p->nchunk * p->D + d_first) * p->N;
            ssm_combine<RN, VEC>(h[k], p->sum_p + at, p->sum_s + at, (long long)p->D * p->N, chunk, (has ? ch : 0) * (unsigned)p->N, nn[k]);
#pragma unroll
            for (int j = 0; j < RN; ++j) h[k][j] = j < count(k) ? h[k][j] : 0.0f;
        }
    }
    const T* pB = (const T*)p->Bm + b * p->b_sb + g * p->b_sg;
    const T* pC = (const T*)p->Cm + b * p->c_sb + g * p->c_sg;
    const uint8_t* ps = p->starts ? p->starts + b * p->starts_sb : nullptr;
    const bool clean = left >= 16 && p->N == 4 * RN * NG;              // every lane's channels and states exist
    float dt_sum = 0.0f;
    bool cut = false;                                   // a start inside the chunk: nothing from before reaches its end

    RawVec<T, 4> nu, nd, nz;
    RawVec<T, RN> nB[NG], nC[NG];
    unsigned nst = 0;
    auto fetch = [&](int tile) {                        // rows behind the length read the last one
        const long long t0 = (long long)tile * kTile;
        const int last = len - 1 - (int)t0, r = row < last ? row : last, rn = ch < last ? ch : last;
        nu = lane_load<T, 4, VEC>(pu + t0 * p->u_st, r * (unsigned)p->u_st, cc);
        nd = lane_load<T, 4, VEC>(pd + t0 * p->dt_st, r * (unsigned)p->dt_st, cc);
        if (!SUMMARY && pz) nz = lane_load<T, 4, VEC>(pz + t0 * p->z_st, r * (unsigned)p->z_st, cc);
#pragma unroll
        for (int k = 0; k < NG; ++k) {                  // lane r of a 16-lane row: step r
            nB[k] = lane_load<T, RN, VEC>(pB + t0 * p->b_st, rn * (unsigned)p->b_st, nn[k]);
            if (!SUMMARY) nC[k] = lane_load<T, RN, VEC>(pC + t0 * p->c_st, rn * (unsigned)p->c_st, nn[k]);
        }
        if (ps) nst = ch <= last ? ps[t0 + rn] : 0;
    };
    const int live = (len + kTile - 1) / kTile, end = tile1 < live ? tile1 : live;      // tiles with a step in them
    if (tile0 < end) fetch(tile0);
    for (int tile = tile0; tile < end; ++tile) {
        const int t0 = tile * kTile;
        const bool plain = clean && t0 + kTile <= len, here = t0 + row < len;
        float u[4], z[4], Bv[NG][RN], Cv[NG][RN];
        float dt[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = (float)nu.v[i];
            dt[i] = (float)nd.v[i] + bias[i];
        }
        if (p->softplus) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float slope;
                dt[i] = softplus_(dt[i], slope);
            }
        }
        if (!SUMMARY && pz) {
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = (float)nz.v[i];
        }
#pragma unroll
        for (int k = 0; k < NG; ++k)
#pragma unroll
            for (int j = 0; j < RN; ++j) { Bv[k][j] = (float)nB[k].v[j]; Cv[k][j] = !SUMMARY ? (float)nC[k].v[j] : 0.0f; }
        if (!plain) {                                   // a step behind the length changes nothing: decay 1, input 0
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                dt[i] = here ? dt[i] : 0.0f;
                u[i] = here ? u[i] : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < NG; ++k)
#pragma unroll
                for (int j = 0; j < RN; ++j) {
                    const bool on = t0 + ch < len && n0(k) + j < p->N;
                    Bv[k][j] = on ? Bv[k][j] : 0.0f;
                    Cv[k][j] = on ? Cv[k][j] : 0.0f;
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s_dt[(c0 + i) * kInLd + row] = dt[i];
            s_du[(c0 + i) * kInLd + row] = dt[i] * u[i];
        }
        const unsigned starts = ps ? ssm_start_bits(nst) : 0u;
        wave_lds_fence();
        if (tile + 1 < end) fetch(tile + 1);
        if (!SUMMARY && p->saved) {
            float* at = p->saved + (((long long)b * p->ntile + tile) * p->D + d_first) * p->N;
#pragma unroll
            for (int k = 0; k < NG; ++k) lane_store<float, RN, VEC>(at, ch * (unsigned)p->N + n0(k), h[k], count(k));
        }
        auto walk = [&](auto with_starts) {
            static_for<4>([&](auto gi) {
                constexpr int tg = decltype(gi)::value * 4;
                const f32x4 dt4 = *(const f32x4*)(s_dt + ch * kInLd + tg), du4 = *(const f32x4*)(s_du + ch * kInLd + tg);
                static_for<4>([&](auto ti) {
                    constexpr int i = decltype(ti)::value, t = tg + i;
                    const bool fresh = decltype(with_starts)::value && ((starts >> t) & 1u);
                    float acc;
#pragma unroll
                    for (int k = 0; k < NG; ++k) {
#pragma unroll
                        for (int j = 0; j < RN; ++j) {
                            const float x = du4[i] * row_bcast<t>(Bv[k][j]);
                            const float hn = __builtin_fmaf(__builtin_amdgcn_exp2f(dt4[i] * A2[k][j]), h[k][j], x);
                            h[k][j] = fresh ? x : hn;
                        }
                        if (!SUMMARY) acc = k == 0 ? dot_row_bcast<t, RN>(Cv[k], h[k]) : acc + dot_row_bcast<t, RN>(Cv[k], h[k]);
                    }
                    if (!SUMMARY) s_y[q * kPartLd + t * 16 + ch] = acc;
                });
                if (SUMMARY) dt_sum += (dt4[0] + dt4[1]) + (dt4[2] + dt4[3]);
            });
        };
        if (starts) { walk(std::true_type{}); cut = true; }
        else walk(std::false_type{});
        wave_lds_fence();
        if (!SUMMARY) {
            f32x4 s = *(const f32x4*)(s_y + row * 16 + c0);
#pragma unroll
            for (int k = 1; k < 4; ++k) s += *(const f32x4*)(s_y + k * kPartLd + row * 16 + c0);
            float out[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = __builtin_fmaf(skip[i], u[i], s[i]);
            if (pz) {
#pragma unroll
                for (int i = 0; i < 4; ++i) out[i] *= z[i] * sigmoidf_(z[i]);
            }
            if (!plain) {
#pragma unroll
                for (int i = 0; i < 4; ++i) out[i] = here ? out[i] : 0.0f;
            }
            lane_store<T, 4, VEC>(py + (long long)t0 * p->D, row * (unsigned)p->D + c0, out, t0 + row < p->T ? nv : 0);
        }
    }
    if (!SUMMARY) {                                     // steps behind the length: zeros
        const float none[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int tile = tile0 > live ? tile0 : live; tile < tile1; ++tile)
            lane_store<T, 4, VEC>(py + (long long)tile * kTile * p->D, row * (unsigned)p->D + c0, none, tile * kTile + row < p->T ? nv : 0);
    }
#pragma unroll
    for (int k = 0; k < NG; ++k) {
        if (SUMMARY) {
            const long long at = (((long long)b * p->nchunk + chunk) * p->D + dch) * p->N + n0(k);
            float P[RN];
#pragma unroll
            for (int j = 0; j < RN; ++j) P[j] = cut ? kCut : __builtin_amdgcn_exp2f(dt_sum * A2[k][j]);
            raw_store<float, RN>(p->sum_p + at, P, count(k), p->vec_n);
            raw_store<float, RN>(p->sum_s + at, h[k], count(k), p->vec_n);
        } else if (p->last && chunk == p->nchunk - 1) {
            raw_store<float, RN>(p->last + ((long long)b * p->D + dch) * p->N + n0(k), h[k], count(k), p->vec_n);
        }
    }
}

// One step.  The state is 8 N bytes per channel of traffic against a few of everything else, so lanes run along it: LPC lanes per channel, four
// states each (16-byte accesses when N % 4 == 0), the sum over the states inside the group of LPC lanes.  A workgroup keeps its A and walks
// batch rows b, b + b_step, ..., the next row's loads in flight while this one is computed.  Bound by memory: 1024 x 1024 channels, N = 16, bf16
// (134 MB of states) take 24.4 us = 5.5 TB/s, the rate of a large copy; one row of 256 channels 2.7 us, a launch.
struct SsmStepParams {
    SsmParams s;
    float* state_out;
    int rows;                          // batch rows a workgroup holds at once (more than 1 when D is small)
    int b_step;
};
template <typename T, int LPC, bool VEC>
__global__ __launch_bounds__(256) void ssm_step_kernel(const SsmStepParams q) {
    const SsmParams& p = q.s;
    const unsigned width = (unsigned)p.D * LPC, flat = blockIdx.x * 256 + threadIdx.x;       // lanes of one batch row
    const unsigned r = q.rows > 1 ? threadIdx.x / width : 0, w = q.rows > 1 ? threadIdx.x - r * width : flat;
    const bool lane_on = q.rows > 1 ? r < (unsigned)q.rows : flat < width;
    const int d = lane_on ? (int)(w / LPC) : 0, k = (int)(w % LPC) * 4, g = d / p.Dg;
    const int n = lane_on ? (p.N - k < 4 ? p.N - k : 4) : 0;
    float A2[4];
    {
        const RawVec<float, 4> A = raw_load<float, 4>(p.A + (long long)d * p.N + k, n, VEC);
#pragma unroll
        for (int j = 0; j < 4; ++j) A2[j] = A.v[j] * kLog2e;
    }
    const float bias = lane_on && p.dt_bias ? p.dt_bias[d] : 0.0f, skip = lane_on && p.Dskip ? p.Dskip[d] : 0.0f;
    struct Row { T u, dt, z; RawVec<T, 4> B, C; RawVec<float, 4> h; bool fresh; } cur, next;
    auto load = [&](Row& x, int b) {
        const bool on = lane_on && b < p.B;
        x.u = on ? ((const T*)p.u)[b * p.u_sb + d] : (T)0.0f;
        x.dt = on ? ((const T*)p.dt)[b * p.dt_sb + d] : (T)0.0f;
        x.z = on && p.z ? ((const T*)p.z)[b * p.z_sb + d] : (T)0.0f;
        x.fresh = on && p.starts && p.starts[b * p.starts_sb];
        x.B = raw_load<T, 4>((const T*)p.Bm + b * p.b_sb + g * p.b_sg + k, on ? n : 0, VEC);
        x.C = raw_load<T, 4>((const T*)p.Cm + b * p.c_sb + g * p.c_sg + k, on ? n : 0, VEC);
        x.h = raw_load<float, 4>(p.state + ((long long)b * p.D + d) * p.N + k, on ? n : 0, VEC);
    };
    int b = blockIdx.y * q.rows + (int)r;
    const int first = blockIdx.y * q.rows;
    load(cur, b);
    for (int b0 = first; b0 < p.B; b0 += q.b_step, b += q.b_step) {
        if (b0 + q.b_step < p.B) load(next, b + q.b_step);
        const float u = (float)cur.u;
        float dt = (float)cur.dt + bias, slope;
        if (p.softplus) dt = softplus_(dt, slope);
        const float du = dt * u;
        float out[4], acc = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float x = du * (float)cur.B.v[j], hn = __builtin_fmaf(__builtin_amdgcn_exp2f(dt * A2[j]), cur.h.v[j], x);
            out[j] = cur.fresh ? x : hn;
            acc = j < n ? __builtin_fmaf((float)cur.C.v[j], out[j], acc) : acc;
        }
        const bool on = lane_on && b < p.B;
        raw_store<float, 4>(q.state_out + ((long long)b * p.D + d) * p.N + k, out, on ? n : 0, VEC);
#pragma unroll
        for (int off = LPC >> 1; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
        if (on && k == 0) {
            acc = __builtin_fmaf(skip, u, acc);
            if (p.z) acc *= (float)cur.z * sigmoidf_((float)cur.z);
            ((T*)p.y)[(long long)b * p.D + d] = (T)acc;
        }
        cur = next;
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------
int ssm_check(const pcrl_ssm_desc* d, const char* who) {
    if (!d) return fail(PCRL_E_ARG, "%s: null descriptor", who);
    if (d->B > (1 << 30) || d->T > 0x7FFFFFE0) return fail(PCRL_E_ARG, "%s: B = %d, T = %d", who, d->B, d->T);      // (a tile's end is a 32-bit step)
    if (d->B < 1 || d->T < 1 || d->D < 1 || d->N < 1 || d->G < 1) return fail(PCRL_E_ARG, "%s: B, T, D, N, G must be positive (%d, %d, %d, %d, %d)", who, d->B, d->T, d->D, d->N, d->G);
    if (d->N > kSsmMaxN) return fail(PCRL_E_ARG, "%s: N = %d states per channel (at most %d)", who, d->N, kSsmMaxN);
    if (d->D % d->G) return fail(PCRL_E_ARG, "%s: %d channels are not shared evenly by %d groups", who, d->D, d->G);
    if (!seq_dtype(d->dtype)) return fail(PCRL_E_ARG, "%s: dtype %d", who, d->dtype);
    for (long long st : {d->u_st, d->dt_st, d->z_st, d->b_st, d->c_st})        // offsets inside a tile of 16 steps are 32-bit
        if (st < 0 || st >= (1LL << 26)) return fail(PCRL_E_ARG, "%s: a step stride of %lld elements (0 to 2^26 - 1)", who, st);
    if (d->D >= (1 << 26)) return fail(PCRL_E_ARG, "%s: D = %d", who, d->D);
    if (!d->u || !d->dt || !d->Bm || !d->Cm || !d->A) return fail(PCRL_E_ARG, "%s: null input", who);
    return PCRL_OK;
}

// One answer for all of them: where B and C admit no whole vectors, the activations are read element by element too.  392 channels, N = 16, B and C
// slices from element 13 of rows of 45, float32, in a graph, us (dense / slices): training pass of 256 x 16 63 / 88, of 4 x 1024 94 / 215; the step's
// own rule below is of the same kind: 1024 rows 17 / 27.
bool ssm_vec(const pcrl_ssm_desc* d, const void* const* extra, const long long* strides, int n_extra) {
    const size_t bytes = 4 * (size_t)elem_bytes(d->dtype);
    if ((d->D / d->G) % 4) return false;
    const void* ptr[3] = {d->u, d->dt, d->z};
    const long long st[3][2] = {{d->u_sb, d->u_st}, {d->dt_sb, d->dt_st}, {d->z_sb, d->z_st}};
    for (int i = 0; i < 3; ++i)
        if (ptr[i] && ((uintptr_t)ptr[i] % bytes || (d->B > 1 && st[i][0] % 4) || (d->T > 1 && st[i][1] % 4))) return false;
    for (int i = 0; i < n_extra; ++i)
        if (extra[i] && ((uintptr_t)extra[i] % bytes || (d->B > 1 && strides[2 * i] % 4) || (d->T > 1 && strides[2 * i + 1] % 4))) return false;
    const int rn = ssm_rn(d->N);
    return d->N % rn == 0 && ((uintptr_t)d->Bm | (uintptr_t)d->Cm) % ((uintptr_t)rn * elem_bytes(d->dtype)) == 0 &&
           ((d->B > 1 ? d->b_sb | d->c_sb : 0) | (d->T > 1 ? d->b_st | d->c_st : 0) | (d->G > 1 ? d->b_sg | d->c_sg : 0)) % rn == 0;
}
bool ssm_vec_n(const pcrl_ssm_desc* d, const void* const* extra, int n_extra) {
    const int rn = ssm_rn(d->N);
    uintptr_t all = (uintptr_t)d->A | (uintptr_t)d->state;
    for (int i = 0; i < n_extra; ++i) all |= (uintptr_t)extra[i];
    return d->N % rn == 0 && all % (4 * (uintptr_t)rn) == 0;
}

void ssm_fill(SsmParams& p, const pcrl_ssm_desc* d) {
    p = SsmParams{};
    p.B = d->B, p.T = d->T, p.D = d->D, p.N = d->N, p.G = d->G, p.Dg = d->D / d->G;
    p.softplus = d->softplus != 0;
    p.ntile = cdiv(d->T, kTile);
    p.u = d->u, p.dt = d->dt, p.z = d->z, p.Bm = d->Bm, p.Cm = d->Cm;
    p.u_sb = d->u_sb, p.u_st = d->u_st, p.dt_sb = d->dt_sb, p.dt_st = d->dt_st, p.z_sb = d->z_sb, p.z_st = d->z_st;
    p.b_sb = d->b_sb, p.b_st = d->b_st, p.b_sg = d->b_sg, p.c_sb = d->c_sb, p.c_st = d->c_st, p.c_sg = d->c_sg;
    p.A = d->A, p.Dskip = d->D_skip, p.dt_bias = d->dt_bias, p.state = d->state;
    p.starts = d->starts, p.starts_sb = d->starts_sb, p.lengths = d->lengths;
}

// How many chunks.  One chunk does the walk's work once; more chunks fill the chip when there are few channel blocks, and pay a summary pass
// (0.4 to 0.7 of the forward's walk, 0.2 to 0.3 of the backward's).  Measured on 16.8 M elements, bf16, N = 16, us (forward / backward, all launches) at 1, 2, 4, 8
// chunks: 128 blocks 321 / 818, 262 / 492, 174 / 343, 152 / 335; 256 blocks 162 / 376, 154 / 329, 140 / 327, -; 384 blocks (25 M elements) 189 / 496,
// 208 / 498, 208 / 482, -; 512 blocks 104 / 268, 126 / 307, 139 / 333, -.  So: none from 1.5 blocks per CU on, else up to 4 workgroups per CU forward
// and 2 backward (its registers and LDS admit no more), down to single tiles (333 steps, 28 blocks: 21 chunks 19 / 33, 11 chunks 21 / 37, 7 chunks 21 / 38).
// Every chunk reads the summaries of all chunks in front of it, and nothing bounds their number: one block of a long sequence pays for that (64
// channels, forward / training pass in a graph, us: 2048 steps 41 / 83, 4096 70 / 143, 8192 -- 512 chunks -- 167 / 323).
SsmPlan ssm_plan(const pcrl_ssm_desc* d, bool backward) {
    SsmPlan plan{};
    const int ntile = cdiv(d->T, kTile);
    plan.nblk = cdiv(d->D / d->G, 64);
    const long long blocks = (long long)d->B * d->G * plan.nblk, cus = num_cus();
    long long chunks = 2 * blocks >= 3 * cus ? 1 : ((backward ? 2 : 4) * cus + blocks - 1) / blocks;
    if (chunks > ntile) chunks = ntile;
    plan.chunk_tiles = cdiv(ntile, chunks);
    plan.nchunk = cdiv(ntile, plan.chunk_tiles);
    return plan;
}

template <typename T, int RN, int NG, bool VEC>
static int launch_fwd(const SsmParams& p, hipStream_t s) {
    const dim3 grid((unsigned)(p.G * p.nblk) * p.nchunk * p.B);
    if (p.nchunk > 1) {
        ssm_fwd_kernel<T, RN, NG, VEC, true><<<grid, 256, 0, s>>>(p);
        PCRL_CHECK_LAUNCH("ssm_fwd_kernel (summary)");
    }
    ssm_fwd_kernel<T, RN, NG, VEC, false><<<grid, 256, 0, s>>>(p);
    PCRL_CHECK_LAUNCH("ssm_fwd_kernel");
    return PCRL_OK;
}
template <typename T, bool VEC>
static int launch_fwd_n(const SsmParams& p, hipStream_t s) {
    return p.N <= 4 ? launch_fwd<T, 1, 1, VEC>(p, s) : p.N <= 8 ? launch_fwd<T, 2, 1, VEC>(p, s) : p.N <= 16 ? launch_fwd<T, 4, 1, VEC>(p, s) : launch_fwd<T, 4, 2, VEC>(p, s);
}
template <typename T>
static int launch_fwd_t(const SsmParams& p, bool vec, hipStream_t s) { return vec ? launch_fwd_n<T, true>(p, s) : launch_fwd_n<T, false>(p, s); }

template <typename T, int LPC>
static void launch_step_n(const SsmStepParams& q, bool vec, dim3 grid, hipStream_t s) {
    if (vec) ssm_step_kernel<T, LPC, true><<<grid, 256, 0, s>>>(q);
    else ssm_step_kernel<T, LPC, false><<<grid, 256, 0, s>>>(q);
}
template <typename T>
static void launch_step(const SsmStepParams& q, int lpc, bool vec, dim3 grid, hipStream_t s) {
    if (lpc == 1) launch_step_n<T, 1>(q, vec, grid, s);
    else if (lpc == 2) launch_step_n<T, 2>(q, vec, grid, s);
    else if (lpc == 4) launch_step_n<T, 4>(q, vec, grid, s);
    else launch_step_n<T, 8>(q, vec, grid, s);
}

static size_t fwd_summary(const pcrl_ssm_desc* d, const SsmPlan& plan) {                 // floats, a multiple of 16 bytes
    return plan.nchunk > 1 ? ((size_t)d->B * plan.nchunk * d->N * d->D + 3) & ~(size_t)3 : 0;
}
static size_t fwd_workspace(const pcrl_ssm_desc* d, const SsmPlan& plan) { return sizeof(float) * 2 * fwd_summary(d, plan); }
size_t ssm_bwd_workspace(const pcrl_ssm_desc* d);       // ssm_bwd.hip

}  // namespace pcrl

using namespace pcrl;

extern "C" int pcrl_ssm_scan_bytes(const pcrl_ssm_desc* d, size_t* workspace, size_t* saved, size_t* bwd) {
    if (int rc = ssm_check(d, "pcrl_ssm_scan_bytes")) return rc;
    if (workspace) *workspace = fwd_workspace(d, ssm_plan(d, false));
    if (saved) *saved = sizeof(float) * (size_t)d->B * cdiv(d->T, kTile) * d->N * d->D;
    if (bwd) *bwd = ssm_bwd_workspace(d);
    return PCRL_OK;
}

extern "C" int pcrl_ssm_scan_fwd(const pcrl_ssm_desc* d, void* y, float* last_state, float* saved, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = ssm_check(d, "pcrl_ssm_scan_fwd")) return rc;
    if (!y) return fail(PCRL_E_ARG, "pcrl_ssm_scan_fwd: null output");
    // (every chunk reads the state, the last one writes last_state)
    if (overlap(last_state, d->state, sizeof(float) * d->B * d->D * d->N, true)) return fail(PCRL_E_ARG, "pcrl_ssm_scan_fwd: last_state overlaps state");
    const SsmPlan plan = ssm_plan(d, false);
    const size_t need = fwd_workspace(d, plan);
    if (need && (!workspace || workspace_bytes < need)) return fail(PCRL_E_WORKSPACE, "pcrl_ssm_scan_fwd: workspace %zu < %zu", workspace_bytes, need);
    if ((long long)d->G * plan.nblk * plan.nchunk * d->B > kMaxGroups) return fail(PCRL_E_ARG, "pcrl_ssm_scan_fwd: too many workgroups");
    SsmParams p;
    ssm_fill(p, d);
    p.nblk = plan.nblk, p.nchunk = plan.nchunk, p.chunk_tiles = plan.chunk_tiles;
    p.y = y, p.last = last_state, p.saved = saved;
    p.sum_p = (float*)workspace, p.sum_s = p.sum_p + fwd_summary(d, plan);
    const void* extra[1] = {y};
    const long long strides[2] = {(long long)d->T * d->D, d->D};
    const void* states[3] = {last_state, saved, workspace};
    p.vec_n = ssm_vec_n(d, states, 3);
    const bool vec = p.vec_n && ssm_vec(d, extra, strides, 1);
    hipStream_t s = (hipStream_t)stream;
    return d->dtype == PCRL_DT_F32 ? launch_fwd_t<float>(p, vec, s) : d->dtype == PCRL_DT_BF16 ? launch_fwd_t<__bf16>(p, vec, s) : launch_fwd_t<_Float16>(p, vec, s);
}

extern "C" int pcrl_ssm_step(const pcrl_ssm_desc* d, void* y, float* state_out, void* stream) {
    if (int rc = ssm_check(d, "pcrl_ssm_step")) return rc;
    if (d->T != 1) return fail(PCRL_E_ARG, "pcrl_ssm_step: T = %d", d->T);
    if (!y || !state_out || !d->state) return fail(PCRL_E_ARG, "pcrl_ssm_step: null output or state");
    if (overlap(state_out, d->state, sizeof(float) * d->B * d->D * d->N, false)) return fail(PCRL_E_ARG, "pcrl_ssm_step: state_out overlaps the state without being it");
    SsmStepParams q;
    ssm_fill(q.s, d);
    q.s.y = y, q.state_out = state_out;
    const int lpc = d->N <= 4 ? 1 : d->N <= 8 ? 2 : d->N <= 16 ? 4 : 8;
    const bool vec = (d->N & 3) == 0 && ((uintptr_t)d->state | (uintptr_t)state_out | (uintptr_t)d->A) % 16 == 0 &&
                     ((uintptr_t)d->Bm | (uintptr_t)d->Cm) % (4 * (uintptr_t)elem_bytes(d->dtype)) == 0 && (d->b_sb | d->b_sg | d->c_sb | d->c_sg) % 4 == 0;
    const long long width = (long long)d->D * lpc;
    if (width > 0x7FFFFFFFLL) return fail(PCRL_E_ARG, "pcrl_ssm_step: D = %d", d->D);
    q.rows = width < 256 ? (int)(256 / width) : 1;
    const unsigned gx = q.rows > 1 ? 1u : (unsigned)cdiv(width, 256), groups = (unsigned)cdiv(d->B, q.rows);
    // workgroups for every row, up to about eight per CU (all resident at once); beyond that each walks several rows
    unsigned gy = (unsigned)((8LL * num_cus() + gx - 1) / gx);
    gy = gy < 1 ? 1 : gy > 65535 ? 65535 : gy;
    gy = gy < groups ? gy : groups;
    q.b_step = (int)gy * q.rows;
    const dim3 grid(gx, gy);
    hipStream_t s = (hipStream_t)stream;
    if (d->dtype == PCRL_DT_F32) launch_step<float>(q, lpc, vec, grid, s);
    else if (d->dtype == PCRL_DT_BF16) launch_step<__bf16>(q, lpc, vec, grid, s);
    else launch_step<_Float16>(q, lpc, vec, grid, s);
    PCRL_CHECK_LAUNCH("ssm_step_kernel");
    return PCRL_OK;
}
