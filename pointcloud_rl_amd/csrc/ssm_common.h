// Selective state space scan: what its forward (ssm_fwd.hip) and backward (ssm_bwd.hip) share.
//
// Work split.  A wave owns all states of 16 channels: lane = 16 q + c holds, of channel c, the RN = ceil(N / 4) states q RN ... q RN + RN - 1 (twice
// that many in two groups for N > 16), so the recurrence runs without any exchange between lanes.  B_t and C_t -- the same for every channel --
// stand in one register per state with step t0 + r in lane r of each 16-lane row, and reach the multiplies as DPP row broadcasts: no scalar
// loads, no LDS.  Steps go by tiles of 16, all of it inside the wave (no workgroup barrier): (1) the 16 x 16 tile of every activation is loaded as
// four adjacent channels per lane, dt and dt u are formed once per element and turned through LDS to four adjacent steps per lane; (2) the 16
// steps are walked; (3) the four state rows' partial sums of each (step, channel) come back through LDS to the loading layout, where they are
// added up, gated and stored.  A workgroup is four such waves on 64 adjacent channels: together they use whole cache lines.
#pragma once
#include "seq_common.h"

namespace pcrl {

constexpr int kTile = 16;              // steps per tile = lanes of a DPP row
constexpr int kSsmMaxN = 32;
constexpr float kCut = -1.0f;          // in the place of a chunk's product of decays (never negative)
constexpr int kInLd = 20;              // [channel][step] tile in LDS: 16-byte reads of four steps, rows 4 banks apart
constexpr int kInTile = 16 * kInLd;
constexpr int kPartLd = 16 * 16 + 16;  // [state row][step][channel]: the four rows of a wave write to different banks
constexpr int kPartTile = 4 * kPartLd;

struct SsmParams {
    int B, T, D, N, G, Dg;             // Dg = D / G channels of a group
    int nblk;                          // blocks of 64 channels per group
    int softplus, vec_n;               // vec_n: the float states admit accesses of RN adjacent states
    int ntile, nchunk, chunk_tiles;    // tiles of the whole sequence; chunks it is cut into, tiles per chunk
    const void *u, *dt, *z, *Bm, *Cm, *dy;
    long long u_sb, u_st, dt_sb, dt_st, z_sb, z_st, b_sb, b_st, b_sg, c_sb, c_st, c_sg, dy_sb, dy_st;
    const float *A, *Dskip, *dt_bias, *state, *dlast;
    const uint8_t* starts; long long starts_sb;
    const int* lengths;
    void* y; float* last; float* saved;            // saved [B][ntile][D][N]: the state in front of each tile
    float* sum_p; float* sum_s;                    // chunk summaries [B][nchunk][D][N]: product of the decays, state from zero
    // backward
    void *du, *ddt, *dz;
    float *part_b, *part_c;                        // [G * nblk][B][T][N]
    float *part_a, *part_d, *part_bias;            // [parts][D][N], [parts][D]
    float* dstate;
    int b_step;                                    // batch rows b, b + b_step, ... share a workgroup
};

// How a call is cut into chunks.
struct SsmPlan { int nblk, nchunk, chunk_tiles; };

int ssm_check(const pcrl_ssm_desc* d, const char* who);
void ssm_fill(SsmParams& p, const pcrl_ssm_desc* d);
SsmPlan ssm_plan(const pcrl_ssm_desc* d, bool backward);
// Whether every access admits whole vectors: four channels of the activations (the extra ones, with their two strides each, included), RN states
// of B, C and the float states (the extra ones included).
bool ssm_vec(const pcrl_ssm_desc* d, const void* const* extra, const long long* strides, int n_extra);
bool ssm_vec_n(const pcrl_ssm_desc* d, const void* const* extra, int n_extra);
__host__ inline int ssm_rn(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : 4; }      // states per lane and group
__host__ inline int cdiv(long long a, long long b) { return (int)((a + b - 1) / b); }

#ifdef __HIPCC__
// The kernel's arguments, read again from the argument segment (scalar loads that hit their cache).  Kept in registers over a tile of a long loop
// they would not fit: the compiler parks them in lanes of vector registers, and every use costs a vector instruction.
typedef const __attribute__((address_space(4))) SsmParams* SsmArgs;
__device__ __forceinline__ SsmArgs ssm_args() {
    SsmArgs a = (SsmArgs)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    return a;
}
// Where this workgroup works: the block index runs channel blocks fastest, then chunks, then batch rows.  Workgroups go to the eight XCDs in
// turn; when they divide evenly, neighbouring ones -- they read the same B_t and C_t -- are dealt to one XCD.
__device__ __forceinline__ void ssm_where(SsmArgs p, int& blk, int& chunk, int& b) {
    const unsigned n = gridDim.x;
    unsigned id = blockIdx.x;
    if ((n & 7u) == 0) id = (id & 7u) * (n >> 3) + (id >> 3);
    const unsigned per = (unsigned)(p->G * p->nblk);
    blk = (int)(id % per);
    const unsigned rest = id / per;
    chunk = (int)(rest % (unsigned)p->nchunk);
    b = (int)(rest / (unsigned)p->nchunk);
}
__device__ __forceinline__ int ssm_length(SsmArgs p, int b) {
    const int* lengths = p->lengths;
    if (!lengths) return p->T;
    const int n = lengths[b];
    return n < 0 ? 0 : n > p->T ? p->T : n;
}
// Bit t: step t0 + t begins a new sequence (steps behind the length never do).  Uniform over the wave.
__device__ __forceinline__ unsigned ssm_start_bits(unsigned char mine) {
    const unsigned long long m = __ballot(mine != 0);
    return (unsigned)__builtin_amdgcn_readfirstlane((int)((unsigned)m & 0xFFFFu));
}
// v = P v + S over n chunk summaries, `step` floats apart (the bases are uniform, `off` and `nn` the lane's clamped place).  Four summaries' loads are
// in flight at a time: the chain is one multiply-add per summary, not one trip to memory.  P == kCut: a start inside
// the chunk, nothing from before gets through (a zero stays one also where the decays' product has overflowed).
template <int RN, bool VEC>
__device__ __forceinline__ void ssm_combine(float (&v)[RN], const float* P, const float* S, long long step, int n, unsigned off, const unsigned (&nn)[RN]) {
    for (int c = 0; c < n; c += 4) {
        RawVec<float, RN> a[4], s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long long at = (c + i < n ? c + i : n - 1) * step;
            a[i] = lane_load<float, RN, VEC>(P + at, off, nn);
            s[i] = lane_load<float, RN, VEC>(S + at, off, nn);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (c + i < n) {
#pragma unroll
                for (int j = 0; j < RN; ++j) v[j] = a[i].v[j] < 0.0f || v[j] == 0.0f ? s[i].v[j] : __builtin_fmaf(a[i].v[j], v[j], s[i].v[j]);
            }
        }
    }
}
// Orders this wave's LDS writes before its LDS reads (LDS executes a wave's accesses in order: only the compiler has to be told).
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
#endif

}  // namespace pcrl
