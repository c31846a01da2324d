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
// Bound by vector instructions (at 16.8 M elements, N = 16: 96 M of a wave's, 23 a state and step, 187 us of every SIMD at 4.3 cycles each; the
// 235 MB it cannot do without would take 44 us) at two waves per SIMD: 256 registers, the states and decays of a tile 128 of them.  More than 8 states
// do not fit them: 8 registers spill in 16 bits and 19 in float32 (26 and 41 where accesses are single elements), 88 to 129 with two state groups.
// Measured at 4 x 2048 x 2048, bf16: 80 us for the chunk summaries, 257 us for the walk, 10 us for the sums.  What was slower for the walk: LDS
// reads one group of steps ahead (302, it spills), states of half a tile at a time (264), the next tile's loads in the middle of the walk (275).
#include "ssm_common.h"

namespace pcrl {

// lo / hi: two values per lane -> one: lanes with the level's bit of their row position clear get lo + partner's lo, the others hi + partner's
// hi.  Partners: position ^ 7 (half-row mirror; first, because it mixes the low bits), ^ 8, ^ 2, ^ 1: after the four levels every position of the
// row is in the sum once.  Levels 0 to 3 settle bits 2, 3, 1, 0 of the position.  The first two -- 12 of the 15 folds of 16 values -- are settled
// by whole 4-lane banks, so that the second addition writes only its banks and no selection is needed: 2 instructions instead of 3.
#define PCRL_FOLD_BANKS(R, LO, HI, CTRL, BANKS)                                           \
    "v_add_f32_dpp %" #R ", %" #LO ", %" #LO " " CTRL " row_mask:0xf bank_mask:0xf\n\t" \
    "v_add_f32_dpp %" #R ", %" #HI ", %" #HI " " CTRL " row_mask:0xf bank_mask:" BANKS "\n\t"
template <int LEVEL, int RN>
__device__ __forceinline__ void fold(float (&out)[RN], const float (&lo)[RN], const float (&hi)[RN], int r) {
    float o[RN];
    if constexpr (LEVEL < 2 && RN == 4) {
        // s_nop 1: the wait states of a DPP read behind the instructions that formed lo and hi
        if constexpr (LEVEL == 0)
            asm("s_nop 1\n\t" PCRL_FOLD_BANKS(0, 4, 8, "row_half_mirror", "0xa") PCRL_FOLD_BANKS(1, 5, 9, "row_half_mirror", "0xa")
                PCRL_FOLD_BANKS(2, 6, 10, "row_half_mirror", "0xa") PCRL_FOLD_BANKS(3, 7, 11, "row_half_mirror", "0xa")
                : "=&v"(o[0]), "=&v"(o[1]), "=&v"(o[2]), "=&v"(o[3]) : "v"(lo[0]), "v"(lo[1]), "v"(lo[2]), "v"(lo[3]), "v"(hi[0]), "v"(hi[1]), "v"(hi[2]), "v"(hi[3]));
        else
            asm("s_nop 1\n\t" PCRL_FOLD_BANKS(0, 4, 8, "row_ror:8", "0xc") PCRL_FOLD_BANKS(1, 5, 9, "row_ror:8", "0xc")
                PCRL_FOLD_BANKS(2, 6, 10, "row_ror:8", "0xc") PCRL_FOLD_BANKS(3, 7, 11, "row_ror:8", "0xc")
                : "=&v"(o[0]), "=&v"(o[1]), "=&v"(o[2]), "=&v"(o[3]) : "v"(lo[0]), "v"(lo[1]), "v"(lo[2]), "v"(lo[3]), "v"(hi[0]), "v"(hi[1]), "v"(hi[2]), "v"(hi[3]));
    } else {
        constexpr int bit = LEVEL == 0 ? 4 : LEVEL == 1 ? 8 : LEVEL == 2 ? 2 : 1;
        const bool up = (r & bit) != 0;
#pragma unroll
        for (int j = 0; j < RN; ++j) {
            const float keep = up ? hi[j] : lo[j], send = up ? lo[j] : hi[j];
            o[j] = keep + dpp_f<LEVEL == 0 ? 0x141 : LEVEL == 1 ? 0x128 : LEVEL == 2 ? 0x4E : 0xB1>(send);
        }
    }
#pragma unroll
    for (int j = 0; j < RN; ++j) out[j] = o[j];
}
// The step whose value a lane at row position r is left with.
__device__ __forceinline__ int folded_step(int r) { return ((r >> 2) & 3) | ((r & 2) << 1) | ((r & 1) << 3); }
// Binary counter of folds: step t = 15 - K arrives; held[l] keeps the upper half of the unfinished pair of level l.  After K = 15 each lane holds in
// held[3] its row's sum of the value of step folded_step(r).
template <int K, int RN>
__device__ __forceinline__ void fold_step(const float (&v)[RN], float (&held)[4][RN], int r) {
    constexpr int t = 15 - K;
    if constexpr ((t & 1) != 0) {
#pragma unroll
        for (int j = 0; j < RN; ++j) held[0][j] = v[j];
    } else if constexpr ((t & 2) != 0) {
        fold<0, RN>(held[1], v, held[0], r);
    } else {
        float f[RN];
        fold<0, RN>(f, v, held[0], r);
        if constexpr ((t & 4) != 0) {
            fold<1, RN>(held[2], f, held[1], r);
        } else {
            fold<1, RN>(f, f, held[1], r);
            if constexpr ((t & 8) != 0) {
                fold<2, RN>(held[3], f, held[2], r);
            } else {
                fold<2, RN>(f, f, held[2], r);
                fold<3, RN>(held[3], f, held[3], r);
            }
        }
    }
}

// LDS per wave, in floats: dt_bias and D of its channels, the three [channel][step] tiles, softplus slopes of the loading layout, three [state row][step][channel] partial sums.
template <bool SUMMARY> constexpr int ssm_bwd_wave_lds() { return SUMMARY ? 32 + 2 * kInTile : 32 + 3 * kInTile + 256 + 3 * kPartTile; }

template <typename T, int RN, int NG, bool VEC, bool SUMMARY>
__global__ __launch_bounds__(256, 2) void ssm_bwd_kernel(const SsmParams) {
    const SsmArgs p = ssm_args();
    constexpr int kWave = ssm_bwd_wave_lds<SUMMARY>();
    extern __shared__ float lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    float* s_bias = lds + wave * kWave;                 // [16], then D [16]
    float* s_dt = s_bias + 32;                          // [channel][step]
    float* s_ds = s_dt + kInTile;
    float* s_du = s_ds + kInTile;
    float* s_slope = s_du + kInTile;
    float* s_gb = s_slope + 256;                        // [state row][step][channel]: sum_n g B
    float* s_aw = s_gb + kPartTile;                     // ... sum_n A w
    float* s_y = s_aw + kPartTile;                      // ... sum_n C h
    float* s_bc = lds + 4 * kWave;                      // [4 waves][dB, dC][16 steps][states of a group]: the four waves' sums over their channels
    int blk, chunk, b0;
    ssm_where(p, blk, chunk, b0);
    if (SUMMARY && chunk == 0) return;                  // nobody ends at the first chunk's summary
    const int g = blk / p->nblk, c_first = (blk - g * p->nblk) * 64 + wave * 16;
    const int left = p->Dg - c_first;                    // channels from this wave's first on; <= 0: it only takes part in the barriers
    if (SUMMARY && left <= 0) return;
    const int d_first = left > 0 ? g * p->Dg + c_first : 0;
    const int tile0 = chunk * p->chunk_tiles, tile1 = tile0 + p->chunk_tiles < p->ntile ? tile0 + p->chunk_tiles : p->ntile;

    const int row = lane >> 2, c0 = (lane & 3) * 4, nv = left - c0 < 4 ? left - c0 : 4;
    unsigned cc[4];
    float d_skip[4], d_bias[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        cc[i] = c0 + i < left ? c0 + i : (VEC || left <= 0 ? 0 : left - 1);
        d_skip[i] = d_bias[i] = 0.0f;
    }
    const int ch = lane & 15, q = lane >> 4, dch = d_first + ch;
    const bool has = ch < left;
    auto n0 = [&](int k) { return (k * 4 + q) * RN; };
    auto count = [&](int k) { const int n = p->N - n0(k); return has ? (n < RN ? n : RN) : 0; };
    unsigned nn[NG][RN];
    float A2[NG][RN], dA[NG][RN];
#pragma unroll
    for (int k = 0; k < NG; ++k) {
        const RawVec<float, RN> a = raw_load<float, RN>(p->A + (long long)dch * p->N + n0(k), count(k), p->vec_n);
#pragma unroll
        for (int j = 0; j < RN; ++j) {
            A2[k][j] = a.v[j] * kLog2e;
            dA[k][j] = 0.0f;
            nn[k][j] = n0(k) + j < p->N ? n0(k) + j : (VEC ? 0 : p->N - 1);
        }
    }
    if (lane < 32) {
        const float* src = lane < 16 ? p->dt_bias : p->Dskip;
        s_bias[lane] = src && has ? src[dch] : 0.0f;
    }
    wave_lds_fence();
    const bool clean = left >= 16 && p->N == 4 * RN * NG;
    const unsigned o_h = (has ? ch : 0) * (unsigned)p->N;

    for (int b = b0; b < p->B; b += p->b_step) {
        const SsmArgs p = ssm_args();
        const int len = ssm_length(p, b);
        const T* pu = (const T*)p->u + b * p->u_sb + d_first;
        const T* pd = (const T*)p->dt + b * p->dt_sb + d_first;
        const T* pz = p->z ? (const T*)p->z + b * p->z_sb + d_first : nullptr;
        const T* pg = (const T*)p->dy + b * p->dy_sb + d_first;
        const T* pB = (const T*)p->Bm + b * p->b_sb + g * p->b_sg;
        const T* pC = (const T*)p->Cm + b * p->c_sb + g * p->c_sg;
        const uint8_t* ps = p->starts ? p->starts + b * p->starts_sb : nullptr;
        const long long obase = (long long)b * p->T * p->D + d_first;           // dense outputs
        float gc[NG][RN];                               // what the steps behind add to g of this one
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            const RawVec<float, RN> l = raw_load<float, RN>(p->dlast + ((long long)b * p->D + dch) * p->N + n0(k), !SUMMARY && p->dlast ? count(k) : 0, p->vec_n);
#pragma unroll
            for (int j = 0; j < RN; ++j) gc[k][j] = l.v[j];
            if (!SUMMARY && chunk < p->nchunk - 1) {     // from the chunks behind, the last one first
                const long long at = (((long long)b * p->nchunk + p->nchunk - 1) * p->D + d_first) * p->N;
                ssm_combine<RN, VEC>(gc[k], p->sum_p + at, p->sum_s + at, -(long long)p->D * p->N, p->nchunk - 1 - chunk, o_h, nn[k]);
#pragma unroll
                for (int j = 0; j < RN; ++j) gc[k][j] = j < count(k) ? gc[k][j] : 0.0f;
            }
        }
        float dt_sum = 0.0f;
        bool cut = false;

        RawVec<T, 4> nu, nd, nz, ng;
        // State groups in flight: all, or (the walk) the next one it comes to; dB and dC leave LDS by the group as well, so that two workgroups fit
        // a CU with two groups too.  N = 32 at 4 x 2048 x 2048: 811 us with both held, 710 with LDS for one, 543 with registers for one.
        constexpr int NF = SUMMARY ? NG : 1;
        RawVec<T, RN> nB[NF], nC[NF];
        RawVec<float, RN> nh[NF];
        unsigned nst = 0;
        auto fetch_states = [&](int tile, int k, int to) {          // rows behind the length read the last one, here and below
            const SsmArgs p = ssm_args();
            const long long t0 = (long long)tile * kTile;
            const int last = len - 1 - (int)t0, rn = ch < last ? ch : last;
            if (!SUMMARY) nB[to] = lane_load<T, RN, VEC>(pB + t0 * p->b_st, rn * (unsigned)p->b_st, nn[k]);
            nC[to] = lane_load<T, RN, VEC>(pC + t0 * p->c_st, rn * (unsigned)p->c_st, nn[k]);
            if (!SUMMARY) nh[to] = lane_load<float, RN, VEC>(p->saved + (((long long)b * p->ntile + tile) * p->D + d_first) * p->N, o_h, nn[k]);
        };
        auto fetch = [&](int tile) {
            const SsmArgs p = ssm_args();
            const long long t0 = (long long)tile * kTile;
            const int last = len - 1 - (int)t0, r = row < last ? row : last, rn = ch < last ? ch : last;
            if (!SUMMARY) nu = lane_load<T, 4, VEC>(pu + t0 * p->u_st, r * (unsigned)p->u_st, cc);
            nd = lane_load<T, 4, VEC>(pd + t0 * p->dt_st, r * (unsigned)p->dt_st, cc);
            if (pz) nz = lane_load<T, 4, VEC>(pz + t0 * p->z_st, r * (unsigned)p->z_st, cc);
            ng = lane_load<T, 4, VEC>(pg + t0 * p->dy_st, r * (unsigned)p->dy_st, cc);
#pragma unroll
            for (int k = 0; k < NF; ++k) fetch_states(tile, k, k);
            if (ps) nst = ch <= last ? ps[t0 + rn] : 0;
        };
        const int live = (len + kTile - 1) / kTile, end = tile1 < live ? tile1 : live;
        if (!SUMMARY) {                                 // steps behind the length: zeros
            const float none[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int tile = tile0 > live ? tile0 : live; tile < tile1; ++tile) {
                const long long at = obase + (long long)tile * kTile * p->D;
                const int n = tile * kTile + row < p->T ? nv : 0;
                const unsigned o = row * (unsigned)p->D + c0;
                lane_store<T, 4, VEC>((T*)p->du + at, o, none, n);
                lane_store<T, 4, VEC>((T*)p->ddt + at, o, none, n);
                if (pz) lane_store<T, 4, VEC>((T*)p->dz + at, o, none, n);
            }
        }
        if (tile0 < end) fetch(end - 1);
        for (int tile = end - 1; tile >= tile0; --tile) {
            const SsmArgs p = ssm_args();
            const int t0 = tile * kTile;
            const bool plain = clean && t0 + kTile <= len, here = t0 + row < len;
            RawVec<T, 4> ru = nu, rz = nz, rg = ng;     // kept as they came: half the registers of a 16-bit type
            float Bv[NG][RN], Cv[NG][RN], h0[NG][RN];
            auto states = [&](int k, int from) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < RN; ++j) {
                    Bv[k][j] = !SUMMARY ? (float)nB[from].v[j] : 0.0f;
                    Cv[k][j] = (float)nC[from].v[j];
                    h0[k][j] = !SUMMARY ? nh[from].v[j] : 0.0f;
                }
                if (!plain) {
#pragma unroll
                    for (int j = 0; j < RN; ++j) {
                        const bool on = t0 + ch < len && n0(k) + j < p->N;
                        Bv[k][j] = on ? Bv[k][j] : 0.0f;
                        Cv[k][j] = on ? Cv[k][j] : 0.0f;
                        h0[k][j] = j < count(k) ? h0[k][j] : 0.0f;
                    }
                }
            };
#pragma unroll
            for (int k = 0; k < NF; ++k) states(k, k);
            if (!plain) {                               // what does not exist counts for nothing (also in the sums over the channels)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool on = here && i < nv;
                    ru.v[i] = on && !SUMMARY ? ru.v[i] : (T)0.0f;
                    rz.v[i] = on && pz ? rz.v[i] : (T)0.0f;
                    rg.v[i] = on ? rg.v[i] : (T)0.0f;
                }
            }
            {
                const f32x4 bias = *(const f32x4*)(s_bias + c0);
                float dt[4], slope[4], ds[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    dt[i] = (float)nd.v[i] + bias[i];
                    ds[i] = (float)rg.v[i];
                    slope[i] = 1.0f;
                }
                if (p->softplus) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) dt[i] = softplus_(dt[i], slope[i]);
                }
                if (pz) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) ds[i] *= (float)rz.v[i] * sigmoidf_((float)rz.v[i]);
                }
                if (!plain) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) dt[i] = here && i < nv ? dt[i] : 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s_dt[(c0 + i) * kInLd + row] = dt[i];
                    s_ds[(c0 + i) * kInLd + row] = ds[i];
                    if (!SUMMARY) {
                        s_du[(c0 + i) * kInLd + row] = dt[i] * (float)ru.v[i];
                        s_slope[i * 64 + lane] = slope[i];
                    }
                }
            }
            const unsigned starts = ps ? ssm_start_bits(nst) : 0u;
            if constexpr (SUMMARY) wave_lds_fence();
            else __syncthreads();                       // the last tile's s_bc has been read
            if (NF < NG) fetch_states(tile, 1, 0);
            else if (tile > tile0) fetch(tile - 1);
            // dB and dC of the tile and of state group k over the workgroup's 64 channels
            constexpr int W = 4 * RN;                   // states of a group as they stand in LDS (N of all exist)
            auto add_bc = [&](int k) __attribute__((always_inline)) {
                const SsmArgs p = ssm_args();
                for (int e = threadIdx.x; e < 2 * 16 * W; e += 256) {
                    const float* src = s_bc + e;
                    const float v = (src[0] + src[2 * 16 * W]) + (src[2 * 2 * 16 * W] + src[3 * 2 * 16 * W]);
                    const int which = e / (16 * W), t = (e / W) % 16, n_ = k * W + e % W;
                    if (n_ < p->N && t0 + t < len) (which ? p->part_c : p->part_b)[(((long long)blk * p->B + b) * p->T + t0 + t) * p->N + n_] = v;
                }
            };
            auto walk = [&](auto with_starts) {
                constexpr bool WS = decltype(with_starts)::value;
                if constexpr (SUMMARY) {
                    static_for<4>([&](auto gi) {
                        constexpr int tg = 12 - decltype(gi)::value * 4;
                        const f32x4 dt4 = *(const f32x4*)(s_dt + ch * kInLd + tg), ds4 = *(const f32x4*)(s_ds + ch * kInLd + tg);
                        static_for<4>([&](auto ti) {
                            constexpr int i = 3 - decltype(ti)::value, t = tg + i;
                            const bool fresh = WS && ((starts >> t) & 1u);
#pragma unroll
                            for (int k = 0; k < NG; ++k) {
                                fma_row_bcast<t, RN>(gc[k], Cv[k], ds4[i]);
#pragma unroll
                                for (int j = 0; j < RN; ++j) {
                                    const float next = gc[k][j] * __builtin_amdgcn_exp2f(dt4[i] * A2[k][j]);
                                    gc[k][j] = fresh ? 0.0f : next;
                                }
                            }
                        });
                        dt_sum += (dt4[0] + dt4[1]) + (dt4[2] + dt4[3]);
                    });
                } else {
                    static_for<NG>([&](auto kc) {
                        constexpr int k = decltype(kc)::value;
                        if (k > 0) {
                            states(k, 0);
                            if (k + 1 < NG) fetch_states(tile, k + 1, 0);
                            else if (tile > tile0) fetch(tile - 1);
                        }
                        float a[kTile][RN], h[kTile][RN];
                        static_for<4>([&](auto gi) {
                            constexpr int tg = decltype(gi)::value * 4;
                            __builtin_amdgcn_sched_barrier(0);       // four steps at a time: interleaving all sixteen spills
                            const f32x4 dt4 = *(const f32x4*)(s_dt + ch * kInLd + tg), du4 = *(const f32x4*)(s_du + ch * kInLd + tg);
                            static_for<4>([&](auto ti) {
                                constexpr int i = decltype(ti)::value, t = tg + i;
                                const bool fresh = WS && ((starts >> t) & 1u);
#pragma unroll
                                for (int j = 0; j < RN; ++j) {
                                    const float x = du4[i] * row_bcast<t>(Bv[k][j]), e = __builtin_amdgcn_exp2f(dt4[i] * A2[k][j]);
                                    const float hn = __builtin_fmaf(e, t == 0 ? h0[k][j] : h[t == 0 ? 0 : t - 1][j], x);
                                    a[t][j] = fresh ? 0.0f : e;
                                    h[t][j] = fresh ? x : hn;
                                }
                                const float acc = dot_row_bcast<t, RN>(Cv[k], h[t]);
                                s_y[q * kPartLd + t * 16 + ch] = k == 0 ? acc : acc + s_y[q * kPartLd + t * 16 + ch];
                            });
                        });
                        asm("" : "+v"(Bv[k][0]));       // broadcast anew on the way back: kept, the 16 copies would take 16 registers
                        float hb[4][RN], hc[4][RN];
                        static_for<4>([&](auto gi) {
                            constexpr int tg = 12 - decltype(gi)::value * 4;
                            __builtin_amdgcn_sched_barrier(0);
                            const f32x4 dt4 = *(const f32x4*)(s_dt + ch * kInLd + tg), du4 = *(const f32x4*)(s_du + ch * kInLd + tg),
                                        ds4 = *(const f32x4*)(s_ds + ch * kInLd + tg);
                            static_for<4>([&](auto ti) {
                                constexpr int i = 3 - decltype(ti)::value, t = tg + i;
                                const bool fresh = WS && ((starts >> t) & 1u);
                                float aw = 0.0f, vb[RN], vc[RN];
                                fma_row_bcast<t, RN>(gc[k], Cv[k], ds4[i]);          // g_t
                                const float gb = dot_row_bcast<t, RN>(Bv[k], gc[k]);
#pragma unroll
                                for (int j = 0; j < RN; ++j) {
                                    vb[j] = gc[k][j] * du4[i];
                                    vc[j] = ds4[i] * h[t][j];
                                    const float gd = gc[k][j] * a[t][j];
                                    float w = gd * (t == 0 ? h0[k][j] : h[t == 0 ? 0 : t - 1][j]);
                                    if (WS) w = fresh ? 0.0f : w;
                                    aw = j == 0 ? w * A2[k][j] : __builtin_fmaf(w, A2[k][j], aw);
                                    dA[k][j] = __builtin_fmaf(w, dt4[i], dA[k][j]);
                                    gc[k][j] = gd;
                                }
                                fold_step<15 - t, RN>(vb, hb, ch);
                                fold_step<15 - t, RN>(vc, hc, ch);
                                const int at = q * kPartLd + t * 16 + ch;
                                s_gb[at] = k == 0 ? gb : gb + s_gb[at];
                                s_aw[at] = k == 0 ? aw : aw + s_aw[at];
                            });
                        });
                        // this wave's sums over its channels, [step][state]: lane (q, ch) has step folded_step(ch), states n0(k) ...
                        float* out = s_bc + wave * (2 * 16 * W) + folded_step(ch) * W + q * RN;
                        if constexpr (RN == 4) {
                            *(f32x4*)out = f32x4{hb[3][0], hb[3][1], hb[3][2], hb[3][3]};
                            *(f32x4*)(out + 16 * W) = f32x4{hc[3][0], hc[3][1], hc[3][2], hc[3][3]};
                        } else {
#pragma unroll
                            for (int j = 0; j < RN; ++j) { out[j] = hb[3][j]; out[16 * W + j] = hc[3][j]; }
                        }
                        if constexpr (k + 1 < NG) {
                            __syncthreads();
                            add_bc(k);
                            __syncthreads();            // before the next group's
                        }
                    });
                }
            };
            if (starts) { walk(std::true_type{}); cut = true; }
            else walk(std::false_type{});
            wave_lds_fence();
            if constexpr (!SUMMARY) {
                const SsmArgs p = ssm_args();
                f32x4 gb = *(const f32x4*)(s_gb + row * 16 + c0), aw = *(const f32x4*)(s_aw + row * 16 + c0), ys = *(const f32x4*)(s_y + row * 16 + c0);
#pragma unroll
                for (int k = 1; k < 4; ++k) {
                    gb += *(const f32x4*)(s_gb + k * kPartLd + row * 16 + c0);
                    aw += *(const f32x4*)(s_aw + k * kPartLd + row * 16 + c0);
                    ys += *(const f32x4*)(s_y + k * kPartLd + row * 16 + c0);
                }
                const f32x4 skip = *(const f32x4*)(s_bias + 16 + c0);
                float o_u[4], o_dt[4], o_z[4], u[4], gy[4], ds[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    u[i] = (float)ru.v[i];
                    ds[i] = gy[i] = (float)rg.v[i];
                }
                if (pz) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float z = (float)rz.v[i], sig = sigmoidf_(z), silu = z * sig;
                        ds[i] = gy[i] * silu;
                        o_z[i] = gy[i] * __builtin_fmaf(skip[i], u[i], ys[i]) * __builtin_fmaf(silu, 1.0f - sig, sig);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    o_u[i] = __builtin_fmaf(s_dt[(c0 + i) * kInLd + row], gb[i], skip[i] * ds[i]);
                    o_dt[i] = __builtin_fmaf(aw[i], kLn2, u[i] * gb[i]) * s_slope[i * 64 + lane];      // the walk summed A log2(e) w
                    d_skip[i] = __builtin_fmaf(ds[i], u[i], d_skip[i]);
                }
                if (!plain) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o_u[i] = here ? o_u[i] : 0.0f;
                        o_dt[i] = here ? o_dt[i] : 0.0f;
                        o_z[i] = here ? o_z[i] : 0.0f;
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) d_bias[i] += o_dt[i];
                const long long to = obase + (long long)t0 * p->D;
                const unsigned o = row * (unsigned)p->D + c0;
                const int n = t0 + row < p->T ? nv : 0;
                lane_store<T, 4, VEC>((T*)p->du + to, o, o_u, n);
                lane_store<T, 4, VEC>((T*)p->ddt + to, o, o_dt, n);
                if (pz) lane_store<T, 4, VEC>((T*)p->dz + to, o, o_z, n);
                __syncthreads();
                add_bc(NG - 1);
            }
        }
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            if (SUMMARY) {
                const long long at = (((long long)b * p->nchunk + chunk) * p->D + dch) * p->N + n0(k);
                float P[RN];
#pragma unroll
                for (int j = 0; j < RN; ++j) P[j] = cut ? kCut : __builtin_amdgcn_exp2f(dt_sum * A2[k][j]);
                raw_store<float, RN>(p->sum_p + at, P, count(k), p->vec_n);
                raw_store<float, RN>(p->sum_s + at, gc[k], count(k), p->vec_n);
            } else if (chunk == 0 && p->dstate) {
                raw_store<float, RN>(p->dstate + ((long long)b * p->D + dch) * p->N + n0(k), gc[k], count(k), p->vec_n);
            }
        }
    }
    if constexpr (!SUMMARY) {
        const SsmArgs p = ssm_args();
        // this wave's part of dA, dD, ddt_bias
        const long long part = (long long)b0 * p->nchunk + chunk;
#pragma unroll
        for (int k = 0; k < NG; ++k) raw_store<float, RN>(p->part_a + (part * p->D + dch) * p->N + n0(k), dA[k], count(k), p->vec_n);
        wave_lds_fence();
#pragma unroll
        for (int i = 0; i < 4; ++i) { s_dt[(c0 + i) * kInLd + row] = d_skip[i]; s_du[(c0 + i) * kInLd + row] = d_bias[i]; }
        wave_lds_fence();
        if (lane < 16 && has) {
            float x = 0.0f, y = 0.0f;
#pragma unroll
            for (int t = 0; t < kTile; ++t) { x += s_dt[ch * kInLd + t]; y += s_du[ch * kInLd + t]; }
            p->part_d[part * p->D + dch] = x;
            p->part_bias[part * p->D + dch] = y;
        }
    }
}

// Adds the parts up in a fixed order.  Workgroups 0 ... n_par - 1: 64 adjacent values of (dA [D][N], dD [D], ddt_bias [D]), 16 threads a value over
// the parts; the others: 1024 elements of dB or dC over the channel blocks of their group.
struct SsmFinishParams {
    int B, T, D, N, G, nblk, parts, n_par;
    const float *part_a, *part_d, *part_bias, *part_b, *part_c;
    float *dA, *dD, *ddt_bias;
    void *dB, *dC;
    const int* lengths;
};
template <typename T>
__global__ __launch_bounds__(1024) void ssm_finish_kernel(const SsmFinishParams p) {
    __shared__ float s_sum[16][64];
    if ((int)blockIdx.x < p.n_par) {
        const long long da = (long long)p.D * p.N, all = da + 2LL * p.D, i = (long long)blockIdx.x * 64 + (threadIdx.x & 63);
        const int k = threadIdx.x >> 6;
        const float* src = i < da ? p.part_a + i : i < da + p.D ? p.part_d + (i - da) : p.part_bias + (i - da - p.D);
        const long long step = i < da ? da : p.D;
        float sum = 0.0f;
        if (i < all) {
#pragma unroll 8
            for (int j = k; j < p.parts; j += 16) sum += src[j * step];
        }
        s_sum[k][threadIdx.x & 63] = sum;
        __syncthreads();
        if (threadIdx.x < 64 && i < all) {
            float t = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j) t += s_sum[j][threadIdx.x];
            if (i < da) p.dA[i] = t;
            else if (i < da + p.D) { if (p.dD) p.dD[i - da] = t; }
            else if (p.ddt_bias) p.ddt_bias[i - da - p.D] = t;
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
// Batch rows that share a workgroup (their dA sums stay in registers, one part of them is left per workgroup): as many as leave about four
// workgroups per CU.  Runs cut into chunks are few rows: one each.
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
size_t ssm_bwd_workspace(const pcrl_ssm_desc* d) { return bwd_layout(d, ssm_plan(d, true)).total; }

template <typename T, int RN, int NG, bool VEC>
static int launch_bwd(const SsmParams& p, hipStream_t s) {
    const dim3 grid((unsigned)(p.G * p.nblk) * p.nchunk * (p.b_step < p.B ? p.b_step : p.B));
    if (p.nchunk > 1) {
        ssm_bwd_kernel<T, RN, NG, VEC, true><<<grid, 256, sizeof(float) * 4 * ssm_bwd_wave_lds<true>(), s>>>(p);
        PCRL_CHECK_LAUNCH("ssm_bwd_kernel (summary)");
    }
    const size_t lds = sizeof(float) * (4 * ssm_bwd_wave_lds<false>() + 4 * 2 * 16 * 4 * RN);
    if (int rc = ensure_dynamic_lds((const void*)ssm_bwd_kernel<T, RN, NG, VEC, false>, lds)) return rc;
    ssm_bwd_kernel<T, RN, NG, VEC, false><<<grid, 256, lds, s>>>(p);
    PCRL_CHECK_LAUNCH("ssm_bwd_kernel");
    return PCRL_OK;
}
template <typename T, bool VEC>
static int launch_bwd_n(const SsmParams& p, hipStream_t s) {
    return p.N <= 4 ? launch_bwd<T, 1, 1, VEC>(p, s) : p.N <= 8 ? launch_bwd<T, 2, 1, VEC>(p, s) : p.N <= 16 ? launch_bwd<T, 4, 1, VEC>(p, s) : launch_bwd<T, 4, 2, VEC>(p, s);
}
template <typename T>
static int launch_bwd_t(const SsmParams& p, bool vec, const SsmFinishParams& f, hipStream_t s) {
    if (int rc = vec ? launch_bwd_n<T, true>(p, s) : launch_bwd_n<T, false>(p, s)) return rc;
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
    if (dy_st < 0 || dy_st >= (1LL << 26)) return fail(PCRL_E_ARG, "pcrl_ssm_scan_bwd: a step stride of %lld elements (0 to 2^26 - 1)", (long long)dy_st);
    const SsmPlan plan = ssm_plan(d, true);
    const BwdLayout at = bwd_layout(d, plan);
    if (!workspace || workspace_bytes < at.total) return fail(PCRL_E_WORKSPACE, "pcrl_ssm_scan_bwd: workspace %zu < %zu", workspace_bytes, at.total);
    const long long elems = 2LL * d->B * d->T * d->G * d->N;
    if ((long long)d->G * plan.nblk * plan.nchunk * d->B > kMaxGroups || elems / 1024 + (long long)d->D * (d->N + 2) / 64 > kMaxGroups / 4 - 2) return fail(PCRL_E_ARG, "pcrl_ssm_scan_bwd: too many workgroups");
    float* w = (float*)workspace;
    SsmParams p;
    ssm_fill(p, d);
    p.nblk = plan.nblk, p.nchunk = plan.nchunk, p.chunk_tiles = plan.chunk_tiles;
    p.b_step = bwd_b_step(d, plan);
    p.saved = const_cast<float*>(saved), p.dy = dy, p.dy_sb = dy_sb, p.dy_st = dy_st, p.dlast = dlast;
    p.du = g->du, p.ddt = g->ddt, p.dz = g->dz, p.dstate = g->dstate;
    p.part_b = w + at.b, p.part_c = w + at.c, p.part_a = w + at.a, p.part_d = w + at.dskip, p.part_bias = w + at.bias;
    p.sum_p = w + at.p, p.sum_s = w + at.s;
    const void* extra[4] = {dy, g->du, g->ddt, g->dz};
    const long long dense[2] = {(long long)d->T * d->D, d->D};
    const long long strides[8] = {dy_sb, dy_st, dense[0], dense[1], dense[0], dense[1], dense[0], dense[1]};
    const void* states[4] = {saved, dlast, g->dstate, workspace};
    p.vec_n = ssm_vec_n(d, states, 4);
    const bool vec = p.vec_n && ssm_vec(d, extra, strides, 4);
    SsmFinishParams f{};
    f.B = d->B, f.T = d->T, f.D = d->D, f.N = d->N, f.G = d->G, f.nblk = plan.nblk, f.parts = p.b_step * plan.nchunk;
    f.n_par = cdiv((long long)d->D * (d->N + 2), 64);
    f.part_a = p.part_a, f.part_d = p.part_d, f.part_bias = p.part_bias, f.part_b = p.part_b, f.part_c = p.part_c;
    f.dA = g->dA, f.dD = g->dD, f.ddt_bias = g->ddt_bias, f.dB = g->dB, f.dC = g->dC, f.lengths = d->lengths;
    hipStream_t s = (hipStream_t)stream;
    return d->dtype == PCRL_DT_F32 ? launch_bwd_t<float>(p, vec, f, s) : d->dtype == PCRL_DT_BF16 ? launch_bwd_t<__bf16>(p, vec, f, s) : launch_bwd_t<_Float16>(p, vec, f, s);
}
