// Selective state space scan: what its forward (ssm_fwd.hip) and backward (ssm_bwd.hip) share.
//
// Work split.  A wave owns 4 of the N states of 64 channels, spread as CPW channels x (64 / CPW) state rows: with CPW = 64 a lane holds 4
// states of one channel, with 32 two, with 16 one.  A workgroup is S = ceil(N / 4) such waves on the SAME CPW channels of one batch row (at
// least 4 waves), so the recurrence runs without any exchange between lanes; B_t and C_t -- the same for every channel -- stand in a register
// per state with step t0 + r in lane r of each 16-lane row, and reach the multiplies as DPP row broadcasts (no scalar loads, no LDS).
// Steps go by tiles of 16: (1) the workgroup loads a 16 x CPW tile, one short vector per thread, forms dt and dt u once and leaves them in
// LDS; (2) every wave walks the 16 steps for its states; (3) the waves' partial sums over the states are added up, gated and stored.
#pragma once
#include "seq_common.h"

namespace pcrl {

constexpr int kTile = 16;              // steps per tile = lanes of a DPP row
constexpr int kSsmMaxN = 32;

struct SsmParams {
    int B, T, D, N, G, Dg;             // Dg = D / G channels of a group
    int S, nblk;                       // waves that hold states; channel blocks per group
    int softplus, vec;                 // vec: every tensor admits whole-vector accesses
    int ntile, nchunk, chunk_tiles;    // tiles of the whole sequence; chunks it is cut into, tiles per chunk
    const void *u, *dt, *z, *Bm, *Cm, *dy;
    long long u_sb, u_st, dt_sb, dt_st, z_sb, z_st, b_sb, b_st, b_sg, c_sb, c_st, c_sg, dy_sb, dy_st;
    const float *A, *Dskip, *dt_bias, *state, *dlast;
    const uint8_t* starts; long long starts_sb;
    const int* lengths;
    void* y; float* last; float* saved;            // saved [B][ntile][N][D]: the state in front of each tile
    float* sum_p; float* sum_s;                    // chunk summaries [B][nchunk][N][D]: product of the decays, state from zero
    // backward
    void *du, *ddt, *dz;
    float *part_b, *part_c;                        // [G * nblk][B][T][N]
    float *part_a, *part_d, *part_bias;            // [parts][N][D], [parts][D]
    float* dstate;
    int parts, b_step;                             // batch rows b, b + b_step, ... share a workgroup
};

// How a call is cut: channels per wave and chunks of the sequence.
struct SsmPlan { int cpw, nblk, nchunk, chunk_tiles; };

int ssm_check(const pcrl_ssm_desc* d, const char* who);
void ssm_fill(SsmParams& p, const pcrl_ssm_desc* d);
SsmPlan ssm_plan(const pcrl_ssm_desc* d);
bool ssm_vec(const pcrl_ssm_desc* d, int V, const void* const* extra, const long long* strides, int n_extra);

__host__ inline int ssm_waves(int N) { return N <= 16 ? 4 : (N + 3) / 4; }
__host__ inline int cdiv(long long a, long long b) { return (int)((a + b - 1) / b); }

#ifdef __HIPCC__
// Where this workgroup works: the block index runs channel blocks fastest, then chunks, then batch rows.  Blocks go to the eight XCDs in turn;
// when a row of channel blocks divides evenly, neighbouring blocks -- they read parts of the same cache lines and the same B_t, C_t -- are
// dealt to one XCD.
__device__ __forceinline__ void ssm_where(const SsmParams& p, int& blk, int& chunk, int& b) {
    const unsigned n = gridDim.x;
    unsigned id = blockIdx.x;
    if ((n & 7u) == 0) id = (id & 7u) * (n >> 3) + (id >> 3);
    const unsigned per = (unsigned)(p.G * p.nblk);
    blk = (int)(id % per);
    const unsigned rest = id / per;
    chunk = (int)(rest % (unsigned)p.nchunk);
    b = (int)(rest / (unsigned)p.nchunk);
}
__device__ __forceinline__ int ssm_length(const SsmParams& p, int b) {
    if (!p.lengths) return p.T;
    const int n = p.lengths[b];
    return n < 0 ? 0 : n > p.T ? p.T : n;
}
// Bit t: step t0 + t begins a new sequence (steps behind the length never do).  Uniform over the wave.
__device__ __forceinline__ unsigned ssm_start_bits(unsigned char mine) {
    const unsigned long long m = __ballot(mine != 0);
    return (unsigned)__builtin_amdgcn_readfirstlane((int)((unsigned)m & 0xFFFFu));
}
#endif

}  // namespace pcrl
